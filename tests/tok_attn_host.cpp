// Attention's kernels built for the CPU: every address that a call touches, in memory and in LDS, lies inside its
// buffers.
#include "host_hip.h"

#include "pcd_reg_hregnet_amd/csrc/tok_attn.hip"

struct Case {
    int B, Nq, Nk, H, Hk, D, causal, kl, ql, mask, buckets, far, both;
};
// kl, ql: lengths that differ by entry (0, one, a part, all and more); mask 2: one for all entries
static const Case cases[] = {
    {1, 1, 1, 1, 1, 8, 0, 0, 0, 0, 0, 0, 0},       {2, 37, 37, 4, 2, 64, 1, 0, 0, 0, 0, 0, 0},
    {2, 1, 200, 4, 1, 128, 1, 1, 0, 0, 0, 0, 0},   {1, 130, 257, 2, 2, 40, 0, 0, 0, 0, 0, 0, 0},
    {3, 65, 33, 6, 2, 32, 1, 1, 0, 0, 0, 0, 0},    {4, 40, 70, 2, 1, 24, 0, 1, 1, 0, 0, 0, 0},
    {4, 40, 70, 2, 1, 72, 1, 1, 1, 1, 0, 0, 0},    {2, 140, 129, 2, 2, 128, 0, 0, 0, 0, 16, 20, 1},
    {1, 161, 161, 3, 3, 64, 1, 0, 0, 0, 32, 128, 0}, {2, 50, 300, 4, 2, 16, 1, 1, 0, 0, 8, 5, 0},
    {2, 150, 50, 2, 2, 80, 0, 1, 1, 2, 4, 2, 1},   {1, 200, 200, 1, 1, 32, 1, 0, 0, 1, 32, 100, 1},
    {1, 2, 700, 2, 1, 48, 0, 0, 0, 0, 128, 1024, 1}, {2, 5, 1030, 8, 2, 128, 1, 1, 0, 1, 32, 128, 0},
    {4, 20, 150, 32, 8, 16, 1, 0, 0, 0, 0, 0, 0},  {1, 133, 140, 6, 1, 8, 0, 0, 1, 1, 8, 30, 1},
    {2, 1, 333, 40, 1, 64, 1, 1, 0, 0, 16, 40, 0}, {1, 2, 100, 64, 2, 32, 0, 0, 0, 0, 32, 1024, 1},
    {2, 70, 150, 4, 2, 96, 1, 1, 0, 0, 0, 0, 0},   {1, 75, 75, 4, 1, 104, 1, 0, 0, 0, 0, 0, 0},
    {2, 3, 400, 8, 2, 88, 1, 1, 0, 0, 32, 128, 0}, {20, 40, 35, 8, 2, 48, 1, 0, 1, 0, 0, 0, 0},
    {20, 33, 129, 8, 2, 88, 0, 1, 0, 2, 16, 20, 1}, {20, 35, 40, 8, 8, 56, 1, 1, 1, 1, 4, 1024, 0},
    {20, 33, 40, 8, 8, 128, 0, 0, 0, 0, 4, 1024, 1}, {3, 4, 9, 2, 1, 64, 1, 1, 1, 1, 64, 64, 1},
    // one row less than whole tiles of 32, 64 and 128 at whole widths
    {2, 63, 63, 2, 2, 64, 0, 0, 0, 0, 0, 0, 0},    {1, 127, 31, 2, 1, 32, 0, 0, 0, 0, 16, 20, 1},
    {20, 31, 63, 8, 8, 128, 1, 0, 0, 0, 0, 0, 0},  {2, 95, 127, 2, 1, 128, 0, 0, 0, 0, 0, 0, 0},
};

static int run(const Case &c, int type, int form) {  // form: which gradients are asked for
    static Guarded g[32];
    int at = 0;
    auto take = [&](size_t bytes, size_t align = 16) { return g[at++].take(bytes, align); };
    const size_t e = type == HREG_TOK_F32 ? 4 : 2;
    hreg_tok_attn_t p = {};
    p.dtype = type, p.B = c.B, p.Nq = c.Nq, p.Nk = c.Nk, p.H = c.H, p.Hk = c.Hk, p.D = c.D, p.causal = p.align_end = c.causal;
    p.scale = 0.125f;
    // rows packed (batch, token, head), or (form 1) heads before tokens with a gap behind each row
    auto rows = [&](int n, int h, int64_t (&s)[3]) {
        const int64_t d = form == 1 ? c.D + 8 : c.D;
        s[0] = (int64_t)n * h * d, s[1] = form == 1 ? d : h * d, s[2] = form == 1 ? n * d : d;
        const size_t last = ((c.B - 1) * s[0] + (n - 1) * s[1] + (h - 1) * s[2] + c.D) * e;
        void *m = take(last);
        for (size_t i = 0; i < last / e; ++i)  // (small numbers: nothing depends on them)
            type == HREG_TOK_F32 ? static_cast<float *>(m)[i] = 0.25f : (float)(static_cast<__bf16 *>(m)[i] = (__bf16)0.25f);
        return m;
    };
    p.q = rows(c.Nq, c.H, p.qs), p.k = rows(c.Nk, c.Hk, p.ks), p.v = rows(c.Nk, c.Hk, p.vs), p.out = rows(c.Nq, c.H, p.os);
    const size_t nq = e * c.B * c.Nq * c.H * c.D, nk = e * c.B * c.Nk * c.Hk * c.D;
    const bool train = form != 3;
    p.lse = train ? static_cast<float *>(take((size_t)8 * c.B * c.H * c.Nq, 4)) : nullptr;
    p.out_rest = train && type == HREG_TOK_BF16 ? take(nq) : nullptr;
    int32_t *kl = static_cast<int32_t *>(take(4 * c.B, 4)), *ql = static_cast<int32_t *>(take(4 * c.B, 4));
    const int part[5] = {100, 60, 0, -1, 300};
    for (int b = 0; b < c.B; ++b) {
        kl[b] = part[(b + form) % 5] < 0 ? 1 : c.Nk * part[(b + form) % 5] / 100;
        ql[b] = part[(b + 1) % 5] < 0 ? 1 : c.Nq * part[(b + 1) % 5] / 100;
    }
    p.k_len = c.kl ? kl : nullptr, p.q_len = c.ql ? ql : nullptr;
    if (c.mask) {
        const int n = c.mask == 2 ? 1 : c.B;
        uint8_t *m = static_cast<uint8_t *>(take((size_t)n * c.Nk, 1));
        for (int i = 0; i < n * c.Nk; ++i) m[i] = i % 7 != 3 && i % 200 < 130;
        p.key_mask = m, p.mask_sb = n == 1 ? 0 : c.Nk;
    }
    if (c.buckets) {
        p.bias_dtype = type;
        void *m = take(e * c.buckets * c.H, e);
        memset(m, 0, e * c.buckets * c.H);
        p.bias = m;
        p.num_buckets = c.buckets, p.max_distance = c.far, p.both = c.both;
        const int side = c.both ? c.buckets / 2 : c.buckets, exact = side / 2;
        p.nthresh = side - exact - 1;
        for (int t = 0; t < p.nthresh; ++t) p.thresh[t] = min(exact + 1 + t * (c.far - exact) / side, c.far);
    }
    auto work = [&](int back) {
        p.ws_bytes = hreg_tok_attn_ws_bytes(&p, back);
        p.ws = p.ws_bytes ? g[30].take((p.ws_bytes + 255) / 256 * 256, 256) : nullptr;
    };
    work(0);
    if (hreg_tok_attn_fwd(&p, nullptr) != HREG_OK) return 1;
    if (!train) return 0;
    p.dout = rows(c.Nq, c.H, p.dos);
    p.dq = form != 2 ? take(nq) : nullptr;
    p.dk = take(nk), p.dv = take(nk);
    p.dbias = c.buckets && form != 2 ? take(e * c.buckets * c.H, e) : nullptr;
    work(1);
    return hreg_tok_attn_bwd(&p, nullptr) != HREG_OK;
}

int main() {
    name_faults();
    int calls = 0;
    for (const Case &c : cases)
        for (int type = 0; type < 2; ++type)
            for (const int form : {0, 1 + (int)(&c - cases + type) % 3}) {
                snprintf(now, sizeof now, "type %d, form %d: %d x %d queries, %d keys, %d heads on %d, width %d, causal %d, lengths %d %d, "
                         "mask %d, buckets %d to %d", type, form, c.B, c.Nq, c.Nk, c.H, c.Hk, c.D, c.causal, c.kl, c.ql, c.mask,
                         c.buckets, c.far);
                if (run(c, type, form)) {
                    printf("refused: %s\n", now);
                    return 2;
                }
                ++calls;
            }
    printf("%d calls inside their buffers\n", calls);
    return 0;
}
