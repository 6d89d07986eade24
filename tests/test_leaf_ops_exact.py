"""Operators over a tree's leaves at the sizes of long and cut leaves, where bounds on rounded sums
say little: operands are small whole numbers, so every sum in any order is exact in 32 bits (below
2^24 in size), and results are compared for equality, 16-bit ones after one rounding. Sums of
float32 rows, held in 64 bits, are compared with random operands too."""

import pytest
import torch

from mpitree_amd import leaf_embedding, leaf_linear, leaf_route
from mpitree_amd.ops import native

TYPES = [torch.float32, torch.float16, torch.bfloat16]
KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def whole(g, shape, dtype, most=2):
    return torch.randint(-most, most + 1, shape, generator=g, device=g.device).to(dtype)


# --------------------------------------------------------------------------- embedding
def run_shift(n, D, dtype):
    """log2 of the sorted rows of a chunk of the table's gradient, for aligned contiguous rows (the
    rule of ``le_run_shift``), checked against the scratch, which is for the shortest chunks that
    any alignment gives."""
    elem = dtype.itemsize

    def shift_of(width):  # elements a lane
        vecs, lanes = -(-D // width), 0
        while lanes < 6 and 1 << lanes < vecs:
            lanes += 1
        blocks, shift = -(-vecs // (1 << lanes)), 8
        least = 4096 if width * elem >= 16 else 2048
        while shift > 4 and (((n >> shift) * blocks) << lanes) // 64 < least:
            shift -= 1
        return shift

    shortest = min(shift_of(w) for w in (8, 4, 2, 1))
    row = 2 * D * (8 if elem == 4 else 4) + 4
    assert native.hip().leaf_embed_grad_bytes(KIND[dtype], n, 1, D, True) == \
        ((n >> shortest) + 1) * row
    return shift_of(next(b // elem for b in (16, 4, elem) if b >= elem and D % (b // elem) == 0))


def cut_leaves(n, chunk, first):
    """n leaf numbers: ``first`` rows of leaf 0, then leaves whose sizes put their ends before, on
    and behind the cuts, leaves of several chunks, leaves of one row and none; shuffled, some rows
    without a leaf."""
    sizes, i, left = [first], 0, n - first
    pattern = [chunk - 1, 1, chunk, chunk + 1, 0, chunk - 1, 2, 3 * chunk, 2 * chunk + 1, 1, 1,
               5 * chunk - 2, chunk // 2, 7]
    while left > 0:
        sizes.append(min(left, pattern[i % len(pattern)]))
        left -= sizes[-1]
        i += 1
    ids = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes)).cuda()
    ids = ids[torch.randperm(n, generator=gen(n + first), device="cuda")]
    return ids, len(sizes) + 3


def table_gradient(ids, G, dy, **kw):
    t = torch.zeros(G, dy.shape[1], dtype=dy.dtype, device="cuda", requires_grad=True)
    (dt,) = torch.autograd.grad(leaf_embedding(ids, t, **kw), t, dy)
    return dt


def sums64(ids, G, dy):
    """Sums by leaf in 64 bits (exact here), a block of columns at a time."""
    if G <= 8:  # (adds of one address one after the other take seconds)
        return torch.stack([dy[ids == q].double().sum(0) for q in range(G)])
    out = torch.zeros(G + 1, dy.shape[1], dtype=torch.float64, device=dy.device)
    key = torch.where((ids >= 0) & (ids < G), ids, G)
    for a in range(0, dy.shape[1], 64):
        out[:, a : a + 64].index_add_(0, key, dy[:, a : a + 64].double())
    return out[:G]


# chunks of 16, 32, ... 256 rows, of narrow and of 16-byte vectors
@pytest.mark.gpu
@pytest.mark.parametrize("n,D,dtype,shift", [
    (9000, 63, torch.float32, 4), (70_000, 63, torch.float32, 5), (140_001, 63, torch.float32, 6),
    (300_000, 63, torch.float32, 7), (1_000_000, 63, torch.float32, 8),
    (300_000, 64, torch.float32, 4), (1_000_003, 64, torch.float32, 5),
    (400_000, 200, torch.float32, 6), (300_001, 512, torch.float32, 7),
    (600_000, 512, torch.float32, 8),
    (100_000, 1024, torch.float16, 5), (200_000, 1024, torch.float16, 6),
    (200_000, 2048, torch.bfloat16, 7), (300_001, 2048, torch.float16, 8),
    (300_000, 62, torch.bfloat16, 6), (600_000, 77, torch.float16, 8)])
@pytest.mark.parametrize("first", [0, 1, 5])
def test_table_gradient_at_the_cuts(n, D, dtype, shift, first):
    assert run_shift(n, D, dtype) == shift
    ids, G = cut_leaves(n, 1 << shift, first)
    g = gen(n + D)
    ids[torch.randint(0, n, (n // 50,), generator=g, device="cuda")] = -1
    dy = whole(g, (n, D), dtype)
    want = sums64(ids, G, dy)
    assert torch.equal(table_gradient(ids, G, dy, scale=0.5), (want * 0.5).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("n,G,D,dtype", [(1_000_000, 1, 63, torch.float32),
                                         (1_000_000, 3, 64, torch.float32),
                                         (1_000_000, 64, 63, torch.float32),
                                         (500_000, 2, 1024, torch.bfloat16),
                                         (500_000, 1, 40, torch.float16)])
def test_table_gradient_of_very_long_leaves(n, G, D, dtype):
    g = gen(n + G)
    ids = torch.randint(-1, G, (n,), generator=g, device="cuda")
    dy = whole(g, (n, D), dtype)
    got, want = table_gradient(ids, G, dy), sums64(ids, G, dy)
    assert torch.equal(got, want.to(dtype))
    assert torch.equal(table_gradient(leaf_route(ids, G), G, dy), got)


def check_sum64(got, want, mass, terms):
    """float32 results of sums held in 64 bits: each of the `terms` additions rounds by at most
    2^-53 of a partial sum, which the absolute sum bounds, and the result is rounded by 2^-24."""
    bound = want.abs() * 2.0 ** -24 + (terms + 2) * 2.0 ** -53 * mass * 2
    off = (got.double() - want).abs() - bound
    assert (off <= 0).all(), float(off.max())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("n,G,D", [(700, 3, 5), (40_000, 2, 63), (200_000, 7, 24), (60_000, 1, 1)])
def test_float32_sums_are_held_in_64_bits(device, n, G, D):
    # sums that cancel to far less than their terms show every lost bit
    g = gen(n, device)
    ids = torch.randint(0, G, (n,), generator=g, device=device)
    dy = torch.randn(n, D, generator=g, device=device)
    dy[n // 2 :] -= dy[: n - n // 2].flip(0) * 0.999
    want, mass = sums64(ids, G, dy), sums64(ids, G, dy.abs())
    t = torch.zeros(G, D, device=device, requires_grad=True)
    (dt,) = torch.autograd.grad(leaf_embedding(ids, t, scale=0.25), t, dy)
    check_sum64(dt, want * 0.25, mass * 0.25, n)
    x = torch.randn(n, 8, generator=g, device=device)
    w, b = (torch.zeros(*s, device=device, requires_grad=True) for s in ((G, D, 8), (G, D)))
    for wrt in ((w, b), (b,)):  # the bias's sums beside dW, and alone
        db = torch.autograd.grad(leaf_linear(x, ids, w, b), wrt, dy)[-1]
        check_sum64(db, want, mass, n)


# ------------------------------------------------------------------------------ linear
def linear_exact(dtype, ids, G, K, N, seed, shift=0, far=0, poison=None):
    """y, dx, dW and db for equality. shift: rows of x and dy start that many elements behind an
    aligned address; far: elements between them, for x and dy in one buffer. poison: NaN beside the
    rows of x and dy (that many columns), in rows without a leaf and in matrices without rows."""
    g, n = gen(seed), ids.numel()
    if far:
        big = torch.empty(n * far, device="cuda", dtype=dtype)
        x = torch.as_strided(big, (n, K), (far, 1))
        dy = torch.as_strided(big, (n, N), (far, 1), 2048)
        x.copy_(whole(g, (n, K), dtype))
        dy.copy_(whole(g, (n, N), dtype))
    else:
        x = whole(g, (n, K + shift), dtype)[:, shift:]
        dy = whole(g, (n, N + shift), dtype)[:, shift:]
    w, b = whole(g, (G, N, K), dtype), whole(g, (G, N), dtype, 9)
    if poison is not None:
        x, dy = (torch.cat([t, torch.full((n, poison), float("nan"), device="cuda", dtype=dtype)],
                           1)[:, : t.shape[1]] for t in (x, dy))
        gone = (ids < 0) | (ids >= G)
        x[gone] = dy[gone] = float("nan")
        met = torch.zeros(G, dtype=torch.bool, device="cuda")
        met[ids[~gone].long()] = True
        w[~met] = b[~met] = float("nan")
    for p in (x, w, b):
        p.requires_grad_()
    y = leaf_linear(x, ids, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x, w, b, y = x.detach(), w.detach(), b.detach(), y.detach()
    seen = torch.zeros(n, dtype=torch.bool, device="cuda")
    for q in torch.unique(ids).tolist():
        if not 0 <= q < G:
            continue
        r = torch.nonzero(ids == q).flatten()
        seen[r] = True
        X, W, D = x[r].double(), w[q].double(), dy[r].double()
        for got, want, what in ((y[r], torch.mm(X, W.t().contiguous()) + b[q].double(), "y"),
                                (dx[r], torch.mm(D, W), "dx"),
                                (dw[q], torch.mm(D.t().contiguous(), X), "dw"),
                                (db[q], D.sum(0), "db")):
            assert want.abs().max() < 2 ** 24
            assert torch.equal(got, want.to(dtype)), (what, q, len(r))
    assert not y[~seen].any() and not dx[~seen].any()
    rest = torch.ones(G, dtype=torch.bool, device="cuda")
    rest[ids[seen]] = False
    assert not dw[rest].any() and not db[rest].any()


def skewed(n, G, skew, none, seed=0):
    g = gen(seed + n + G)
    p = (torch.arange(G, dtype=torch.float64, device="cuda") + 1) ** -skew
    ids = torch.searchsorted(torch.cumsum(p / p.sum(), 0),
                             torch.rand(n, generator=g, device="cuda", dtype=torch.float64))
    ids = torch.randperm(G, generator=g, device="cuda")[ids.clamp(max=G - 1)]
    ids[torch.rand(n, generator=g, device="cuda") < none] = -1
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,K,N,skew", [
    (40_000, 9, 24, 20, 2.5), (40_000, 9, 24, 20, 0.0), (200_000, 1, 64, 64, 0.0),
    (200_000, 3, 32, 1, 0.5), (100_000, 2500, 64, 48, 1.5), (100_000, 700, 32, 24, 1.0),
    (60_000, 5, 33, 130, 1.0)])
def test_long_and_cut_leaves(dtype, n, G, K, N, skew):
    linear_exact(dtype, skewed(n, G, skew, 0.05), G, K, N, n + K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,K,N,skew,shift", [
    (66_000, 5, 520, 776, 0.5, 0), (33_000, 23, 1048, 1032, 1.0, 0),
    (16_500, 16, 1023, 1029, 0.0, 0),  # the largest tiles in all directions, from packed operands
    (16_500, 16, 1023, 1029, 0.5, 3), (16_500, 16, 1024, 1032, 0.5, 8),
    (20_000, 7, 523, 1001, 0.0, 0), (12_000, 300, 520, 777, 0.0, 0)])
def test_large_products(dtype, n, G, K, N, skew, shift):
    linear_exact(dtype, skewed(n, G, skew, 0.02), G, K, N, n + K, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,used,K,N", [(16_384, 4096, 8, 256, 264), (5000, 2000, 3, 64, 40),
                                          (9000, 20_000, 2, 24, 16), (70, 50_000, 5, 16, 8)])
def test_rows_in_few_of_many_leaves(dtype, n, G, used, K, N):
    # the mean rows of a leaf say nothing of the leaves that have some
    g = gen(n)
    some = torch.randperm(G, generator=g, device="cuda")[:used]
    ids = some[torch.randint(0, used, (n,), generator=g, device="cuda")]
    linear_exact(dtype, ids, G, K, N, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_rows(dtype):
    # rows so far apart that their last offsets pass 2^32 elements
    n, G, K, N = 8400, 3, 1800, 1816
    linear_exact(dtype, skewed(n, G, 0.0, 0.1), G, K, N, 61, far=2 ** 32 // n // 8 * 8 + 4096)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [40, 700, 30_000])
def test_rows_that_are_one_row(dtype, n):
    # an input row and an incoming gradient that are broadcast over the rows
    g, G, K, N = gen(n), 5, 72, 48
    ids = torch.randint(-1, G, (n,), generator=g, device="cuda", dtype=torch.int32)
    one, d1 = whole(g, (1, K), dtype), whole(g, (1, N), dtype)
    w, b = whole(g, (G, N, K), dtype), whole(g, (G, N), dtype)
    p = one.clone().requires_grad_()
    for t in (w, b):
        t.requires_grad_()
    y = leaf_linear(p.expand(n, K), ids, w, b)
    dp, dw, db = torch.autograd.grad(y, (p, w, b), d1.expand(n, N))
    rows = torch.bincount(ids[ids >= 0].long(), minlength=G)
    W, X, D = w.detach().double(), one.double(), d1.double()
    each = (W * D[:, :, None]).sum(1)  # a row's gradient in each leaf
    assert torch.equal(dw, (rows[:, None, None] * D.t() * X).to(dtype))
    assert torch.equal(db, (rows[:, None] * D).to(dtype))
    # torch sums the rows' gradients (rounded to the type, exact here) in a type of its own choice
    full = (rows[:, None] * each).sum(0)
    assert each.abs().max() < 256  # exact in every type
    mass = (rows[:, None] * each.abs()).sum(0)
    off = (dp[0].double() - full).abs() - full.abs() * torch.finfo(dtype).eps - 2.0 ** -20 * mass
    assert (off <= 0)[mass < torch.finfo(dtype).max].all()
    want = torch.where((ids >= 0)[:, None],
                       ((W * X).sum(2) + b.detach().double())[ids.clamp(min=0).long()], 0.0)
    assert torch.equal(y, want.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,K,N,poison", [
    (50, 9, 40, 24, 8), (64, 100, 33, 17, 1), (3000, 7, 64, 64, 8), (3000, 2500, 64, 48, 8),
    (3000, 90, 13, 21, 3), (5000, 12, 264, 136, 16), (5000, 12, 201, 199, 1), (9000, 3, 32, 1, 7),
    (16_500, 20, 1024, 1032, 8), (16_500, 20, 1023, 1029, 3)])
def test_nan_around_the_operands(dtype, n, G, K, N, poison):
    # nothing that is no operand of a row reaches it, nor what a tile holds behind its end
    linear_exact(dtype, skewed(n, G, 1.0, 0.1), G, K, N, n + K, poison=poison)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,D,pad", [(30, 9, 7, 1), (3000, 50, 63, 5), (20_000, 3, 64, 8),
                                       (9000, 4000, 1024, 8)])
def test_nan_around_a_table_and_its_gradient(dtype, n, G, D, pad):
    g, ids = gen(n), skewed(n, G, 1.0, 0.1)
    dy, t = whole(g, (n, D + pad), dtype), whole(g, (G, D + pad), dtype, 9)
    dy[:, D:], t[:, D:] = float("nan"), float("nan")
    dy[ids < 0] = float("nan")
    want = sums64(ids, G, torch.where((ids < 0)[:, None], 0.0, dy[:, :D]).to(dtype))
    assert torch.equal(table_gradient(ids, G, dy[:, :D]), want.to(dtype))
    y = leaf_embedding(ids, t[:, :D], scale=2.0)
    rows = t[:, :D].double()[ids.clamp(min=0)] * 2.0
    assert torch.equal(y, torch.where((ids < 0)[:, None], 0.0, rows).to(dtype))
