// The block boundary's kernels built for the CPU: every address that a call touches lies inside its buffers.
#include "host_hip.h"

#include "pcd_reg_hregnet_amd/csrc/tok_elem.hip"

int main() {
    name_faults();
    static Guarded g[19];
    int calls = 0;
    // forms of the call: both norms and both gradients (the usual one), an RMS norm before alone, a norm
    // behind alone, the first norm of a stack; the gate for all, for some, for one of the rows, or none
    struct Form { int post, pre, f, bias; };
    const Form forms[] = {{2, 2, 1, 1}, {1, 1, 1, 0}, {0, 1, 1, 0}, {2, 0, 1, 1}, {0, 2, 0, 1}};
    std::vector<int> widths = {2048, 4096, 8191, 8192};  // (one more chunk than a whole row: 1032, 2056, ..)
    for (int C = 1; C <= 8192; C += C < 160 ? 1 : C < 1100 ? 8 : 44) widths.push_back(C);
    for (int C = 1024; C < 8192; C *= 2) widths.push_back(C + 8), widths.push_back(2 * C - 8);
    for (const int C : widths)
        for (int type = 0; type < 2; ++type) {
            const Form fm = forms[(C / 8 + type) % 5];
            for (int k = 0; k < 2; ++k) {
                const Form f = k ? fm : forms[0];
                const int R = C > 512 ? 2 : 6, kind = f.f ? (C / 8 + k) % 4 : 0, rows = kind == 1 ? R : kind == 2 ? R / 2 : 1;
                const int ptype = (C / 8 + type + k) % 2 ? HREG_TOK_F32 : type;
                const size_t e = type == HREG_TOK_F32 ? 4 : 2, pe = ptype == HREG_TOK_F32 ? 4 : 2, n = e * R * C;
                const size_t gn = e * C * (R / rows);
                snprintf(now, sizeof now, "type %d, parameters %d, %d rows of %d, norms %d and %d, gate rows %d, f %d", type, ptype, R,
                         C, f.post, f.pre, kind ? rows : 0, f.f);
                hreg_tok_block_t p = {};
                p.dtype = type, p.param_dtype = ptype, p.R = R, p.C = C, p.gate_rows = rows, p.post = f.post, p.pre = f.pre;
                p.scale = 1.f, p.eps = 1e-6f, p.step = C % 16 ? 0 : 6554, p.seed = 7;
                int at = 0;
                auto take = [&](size_t bytes, size_t align = 16) { return g[at++].take(bytes, align); };
                p.x = take(n);
                p.f = f.f ? take(n) : nullptr;
                p.gate = kind ? take(gn) : nullptr;
                p.post_w = f.post ? take(pe * C) : nullptr;
                p.post_b = f.post && f.bias ? take(pe * C) : nullptr;
                p.pre_w = f.pre ? take(pe * C) : nullptr;
                p.pre_b = f.pre && f.bias ? take(pe * C) : nullptr;
                p.y = f.f ? take(n) : nullptr;
                p.h = f.pre ? take(n) : nullptr;
                p.stats = static_cast<float *>(take(16 * R));
                if (hreg_tok_block_fwd(&p, nullptr) != HREG_OK) return 2;
                if (!f.f) p.y = const_cast<void *>(p.x), p.step = 0;
                p.dy = take(n);
                p.dh = f.pre ? take(n) : nullptr;
                p.dx = take(n);
                p.df = f.f ? take(n) : nullptr;
                p.dgate = kind ? take(gn) : nullptr;
                // (parameters' gradients are as long as the parameters, workspaces end at their size rounded up)
                static Guarded d[4], w;
                p.dpost_w = p.post_w ? d[0].take(pe * C, pe) : nullptr;
                p.dpost_b = p.post_b ? d[1].take(pe * C, pe) : nullptr;
                p.dpre_w = p.pre_w ? d[2].take(pe * C, pe) : nullptr;
                p.dpre_b = p.pre_b ? d[3].take(pe * C, pe) : nullptr;
                p.ws_bytes = hreg_tok_block_ws_bytes(&p);
                p.ws = w.take((p.ws_bytes + 255) / 256 * 256, 256);
                if (hreg_tok_block_bwd(&p, nullptr) != HREG_OK) return 3;
                ++calls;
            }
        }
    printf("%d calls inside their buffers\n", calls);
    return 0;
}
