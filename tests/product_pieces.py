"""Inputs of the cross entropy against a table whose answers lie in the low pieces of float32 products, and what they come to.

Where float32 rows are carried as three bfloat16 pieces each, a product is six of the nine piece products: (0,0), (0,1), (1,0), (1,1),
(0,2), (2,0).  Worst-case bounds of long sums are wider than the last three of them; these cases are made so that leaving out any one
shows.  `product` is the float32 product under test."""
import math

import torch

PAIRS = ((2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0))
# n, V, C: sizes whose 1 / V has a second piece of 2^-9.5 of it and a third of 2^-18.5, at the least
LOW_PIECES = [(300, 119, 130), (257, 811, 65), (700, 3001, 200), (300, 119, 64), (1021, 811, 32)]
MIDDLE, LOW = 1.5 * 2.0 ** -9, 56 * 2.0 ** -23      # of 1 + MIDDLE + LOW: the second piece and the third


def pieces(x):
    out = []
    for _ in range(3):
        p = x.bfloat16().float()
        out.append(p)
        x = x - p
    return out


def product_of(pairs):
    """a @ b.T of float32 matrices, by these piece products, summed in float32."""
    def product(a, b):
        pa, pb = pieces(a), pieces(b)
        total = torch.zeros(a.shape[0], b.shape[0])
        for i, j in pairs:
            total = total + pa[i] @ pb[j].t()
        return total
    return product


# ------------------------------------------------------------------ logits
SCALE = 2.0 ** 20


def logit_case(which, n, V, C):
    """x, weight, and the logits before SCALE, which float32 arithmetic of all piece products reaches exactly: the products of the high
    pieces cancel, and what is left is a third piece, or the product of two second ones, times 0, 1/2 or 1 by table row."""
    x, w = torch.zeros(n, C), torch.zeros(V, C)
    at = [C - 1, 3, C // 2]
    if which == (1, 1):
        left, right, value = (1 + MIDDLE, 1.0, MIDDLE), (1 + MIDDLE, -1 - MIDDLE, -1.0), MIDDLE * MIDDLE
    else:
        left, right, value = (1 + MIDDLE + LOW, 1 + MIDDLE, 0.0), (1.0, -1.0, 0.0), LOW
        if which == (0, 2):
            left, right = right, left
    share = torch.tensor([0.0, 0.5, 1.0])[torch.arange(V) % 3]
    for c, a, b in zip(at, left, right):
        x[:, c], w[:, c] = a, b * share
    return x, w, (value * share).expand(n, V)


# ------------------------------------------------------------------ gradients
def gradient_case(n, V, C):
    """x and weight of disjoint columns: every logit is 0, every probability 1 / V.  Column c of x is 0 but for one row, of the table but
    for one row: an element of either gradient is then one product (1 / V) value, 24 bits of each -- or, where the product is with the
    target's probability, (1 / V - 1) value.  -> x, weight, [(row of the table, row of x, column, value)] for dW, the same for dx."""
    x, w = torch.zeros(n, C), torch.zeros(V, C)
    half = C // 2
    values = torch.tensor([1.0, 1 + MIDDLE, 1 + MIDDLE + LOW, 1 + LOW, 1 - MIDDLE - LOW])
    of_x = [(i * 37 % n, c, float(values[c % 5])) for i, c in enumerate(range(half))]
    of_w = [(i * 11 % V, c, float(values[c % 5])) for i, c in enumerate(range(half, C))]
    for row, c, v in of_x:
        x[row, c] = v
    for row, c, v in of_w:
        w[row, c] = v
    return x, w, of_x, of_w


# 1 / V as float32 reaches it: the logarithm of V (one unit in the last place of a number below 16: 2^-20 in the exponent at worst), an
# exponential (one unit); then the sum's five additions, what the left-out piece products come to (2^-25), and two factors of 1
def gradient_bound(V):
    ulp_of_log = 2.0 ** (math.floor(math.log2(math.log2(V))) - 23)
    return ulp_of_log * math.log(2) + 2.0 ** -23 + (5 + 1 + 2) * 2.0 ** -24


def gradient_errors(V, gx, gw, t, of_x, of_w):
    """Largest relative error of the elements of dx and dW that are one product; t: the rows' targets."""
    p, worst = 1.0 / V, 0.0
    for row, c, v in of_w:      # dx[i][c] = (p - [t_i = row]) v, for every i
        want = (p - (t == row).double()) * v
        worst = max(worst, float(((gx[:, c].double() - want) / want).abs().max()))
    for row, c, v in of_x:      # dW[j][c] = (p - [t_row = j]) v, for every j
        want = torch.full((V,), p, dtype=torch.float64) * v
        want[t[row]] -= v
        worst = max(worst, float(((gw[:, c].double() - want) / want).abs().max()))
    return worst
