"""How near float32 attention has to come to the 64-bit form, over whole tensors (norm of the error by the
norm of the value).  token_oracle.py's bounds are for single elements: they add up the largest error of every
rounding, a thousand times what float32 products lose together.

Errors of different elements are independent of each other, so over a tensor they count by their root mean
square.  In units of 2^-24: a score of D products is made in 6 D / 16 additions (six products of pieces,
sixteen deep), each off by at most 2 of a partial sum that is on average below half of the whole in square;
do . v likewise, but a gradient feels both with weights below one, so the two together are taken as one whole
6 D / 16.  What the left-out piece products add (8 at most, of a product's own size and sign: a factor of the
score), the exponential and its argument (2 each), p's and ds's pieces (8) and 32 rows' product (12 additions,
one of two halves at a time): 36 together.

A sum over many pairs (the bias table's gradient) keeps the relative error of its terms as long as that is
without a sign of its own; a rounding that goes one way grows with the square root of their number.  The
terms' error is the root of the sum of squares, each addition's 1 / sqrt(3) of its largest: sqrt(6 D / 16) *
1.2 twice, and 4 for the rest: below 8 up to 48 columns, and twice that allowed."""

U = 2.0 ** -24


def tolerance(D):
    """for out, dq, dk, dv at up to some hundred keys"""
    return (6 * D / 16 + 36) * U


def tolerance_table(D):
    """for dbias over about 10^6 pairs"""
    assert D <= 48
    return 16 * U


def error(got, value):
    return ((got.double() - value).norm() / value.norm()).item()


SHAPES = [  # B, Nq, Nk, heads, key heads, width, causal, buckets
    (1, 161, 161, 2, 2, 64, True, (32, 128, False)),
    (1, 130, 257, 2, 1, 40, False, None),
    (1, 65, 33, 2, 2, 32, False, None),
    (1, 128, 300, 1, 1, 128, False, (16, 20, True)),
    (1, 20, 20, 1, 1, 8, False, None),
    (2, 1, 400, 4, 2, 64, True, (32, 128, False)),  # rows of a key head in one tile: the keys are split
]
