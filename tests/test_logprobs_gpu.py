"""Log probabilities, entropy and top alternatives against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF = float("inf")


def _ops():
    from sparkpipe_rs_b200 import ops

    return ops


def reference(logits, ids, k):
    """(logprobs, entropy, top logprobs, top ids) in 64 bits, on the CPU."""
    x = logits.double().cpu()
    T, V = x.shape
    bad = (torch.isnan(x) | (x == INF)).any(1)
    m = torch.where(bad, 0.0, x.amax(1))
    empty = ~bad & (m == -INF)
    t = x - torch.where(empty, 0.0, m)[:, None]
    lse = torch.where(empty, 0.0, torch.log(t.exp().sum(1)))
    lp = t - lse[:, None]
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    ent = torch.where(bad, math.nan, torch.where(empty, 0.0, ent))
    i = ids.long().cpu().view(T, -1)
    given = torch.gather(lp, 1, i.clamp(0, V - 1))
    given = torch.where((i < 0) | (i >= V) | bad[:, None], math.nan, given)
    given = torch.where(i == -1, 0.0, given)
    key = torch.where(bad[:, None], -INF, x)
    best = torch.sort(key, dim=1, descending=True, stable=True)
    value, index = best.values[:, :k], best.indices[:, :k]
    top = torch.gather(lp, 1, index)
    none = value == -INF
    top = torch.where(bad[:, None], math.nan, torch.where(none, -INF, top))
    return given.view(ids.shape), ent, top, torch.where(none, -1, index)


def check(out, ref):
    """|t| = |x - m| is one fp32 rounding off (2^-24 |t|) and log p one more. S: each term is
    exp2 of a rounded product (2^-24 |t| log2 e in the exponent, where terms with large |t|
    weigh e^-|t|, so under 2^-23) and exp2's own 2^-22, and at most 2^-20 for the fp32 adds of
    a thread: ln S is within 2^-19 = 1.9e-6 and entropy, a mean of |t| <= ln V + 1 with the
    same weights, within 2^-19 (1 + |H| + 8)."""
    lp, ent, top, ids = [a.cpu() for a in out]
    for got, want in ((lp, ref[0]), (top, ref[2])):
        # the outputs are fp32: a log p below its range (lowest - max / 4 = -1.25 * 2^128) is -inf there
        torch.testing.assert_close(got.double(), want.float().double(), rtol=2**-22, atol=2**-18, equal_nan=True)
    torch.testing.assert_close(ent.double(), ref[1], rtol=2**-18, atol=2**-15, equal_nan=True)
    assert torch.equal(ids.long(), ref[3])


def make(T, V, dtype, seed, pad=0, shift=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(T, V + pad + shift, device=DEV, generator=g) * scale).to(dtype)
    return x[:, shift:shift + V], torch.randint(0, V, (T,), device=DEV, generator=g).int()


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,k,pad,shift", [(1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (2, 7, 3, 5, 1), (5, 31, 0, 0, 0),
                                             (4, 257, 32, 0, 3), (37, 1000, 20, 0, 0), (3, 4099, 5, 1, 1),
                                             (300, 511, 8, 9, 7), (1, 102400, 20, 0, 0), (2, 163840, 32, 0, 0),
                                             (9, 50001, 20, 6, 5), (1025, 2048, 1, 0, 0)])
def test_rows(dtype, T, V, k, pad, shift):
    x, ids = make(T, V, dtype, T * 31 + V, pad, shift)
    check(_ops().token_logprobs(x, ids, top_k=k), reference(x, ids, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,pad,shift", [(1, 8191, 0, 0), (2, 8192, 8, 0), (32, 16385, 0, 0), (33, 16391, 3, 1),
                                           (64, 32767, 2, 5), (65, 32769, 0, 0), (31, 40001, 7, 7)])
def test_rows_around_the_splits(dtype, T, V, pad, shift):
    """Rows and lengths at which a row is one, four or eight CTAs' work, the last of them short."""
    x, ids = make(T, V, dtype, T * 17 + V, pad, shift)
    ids[0], ids[-1] = V - 1, 0
    for k in (0, 32):
        check(_ops().token_logprobs(x, ids, top_k=k), reference(x, ids, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,shift", [(32, 0), (63, 1), (200, 0), (256, 3), (517, 0), (556, 5), (1000, 0), (1091, 2),
                                     (2048, 0), (2111, 63)])
def test_short_rows(dtype, V, shift):
    """Rows of few vectors, where groups of threads are small: whole, masked to a few logits, and with ties."""
    x, ids = make(48, V, dtype, V + shift, 0, shift)
    x = x.clone() if shift == 0 else x
    g = torch.Generator(device=DEV).manual_seed(V)
    x[16:32].masked_fill_(torch.rand(16, V, device=DEV, generator=g) < 0.9, -INF)
    x[32:].copy_(torch.randint(-3, 4, (16, V), device=DEV, generator=g).to(dtype))
    for k in (1, 20, 32):
        check(_ops().token_logprobs(x, ids, top_k=k), reference(x, ids, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,shift", [(601, 31, 0), (700, 300, 1), (640, 1000, 63), (1800, 2049, 5), (1777, 8190, 3)])
def test_many_short_rows(dtype, T, V, shift):
    """More rows than run at once; rows of equal logits, masked ones, one that holds NaN."""
    x, ids = make(T, V, dtype, V + T, 2, shift)
    g = torch.Generator(device=DEV).manual_seed(V)
    x[100:300].masked_fill_(torch.rand(200, V, device=DEV, generator=g) < 0.95, -INF)
    x[300:310] = 1.5
    x[310] = -INF
    x[311, V // 2] = math.nan
    x[400:600].copy_(torch.randint(-3, 4, (200, V), device=DEV, generator=g).to(dtype))
    for k in (0, 5, 31):
        check(_ops().token_logprobs(x, ids, top_k=k), reference(x, ids, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 3001, 102400])
def test_ties_and_order(dtype, V):
    """Equal logits, whole-number logits, rising and falling rows, -0.0 beside 0.0."""
    g = torch.Generator(device=DEV).manual_seed(V)
    col = torch.arange(V, device=DEV, dtype=torch.float32)
    zeros = torch.where(torch.rand(V, device=DEV, generator=g) < 0.5, 0.0, -0.0)
    rows = [torch.full((V,), 1.5, device=DEV), torch.randint(0, 4, (V,), device=DEV, generator=g).float(),
            col * 2**-8, -col * 2**-8, zeros, torch.where(col % 97 == 5, 3.0, -1.0),
            torch.where(col > V - 60, 2.0, 1.0), torch.where(col < 50, 2.0 + col * 2**-5, 0.0)]
    x = torch.stack(rows).to(dtype)
    ids = torch.randint(0, V, (len(rows),), device=DEV, generator=g).int()
    check(_ops().token_logprobs(x, ids, top_k=32), reference(x, ids, 32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [33, 5003, 102400])
def test_masks(dtype, V):
    """Rows that a mask leaves empty or nearly so, the type's lowest value, NaN and +inf."""
    x, _ = make(12, V, dtype, V + 1)
    x = x.clone()
    low = torch.finfo(dtype).min
    x[0] = -INF
    x[1] = -INF
    x[1, V - 1] = 0.5
    x[2] = -INF
    x[2, 3::11] = torch.arange(x[2, 3::11].numel(), device=DEV).to(dtype) % 5
    x[3] = low
    x[4] = low
    x[4, V // 2] = -2.0
    x[5, ::2] = low
    x[6, 7] = INF
    x[7, V - 2] = math.nan
    x[8] = math.nan
    x[9, :] = -INF
    x[9, 4] = math.nan
    x[10] = torch.finfo(dtype).max / 4
    x[10, 5] = low
    x[11, :] = -INF
    x[11, :2] = low
    ids = torch.tensor([[0, V - 1, -1, 5, V, -7]], device=DEV, dtype=torch.int32).expand(12, 6).contiguous()
    check(_ops().token_logprobs(x, ids, top_k=20), reference(x, ids, 20))


@pytest.mark.parametrize("n", [0, 1, 3, 300])
def test_given_tokens(n):
    x, _ = make(6, 999, torch.bfloat16, n)
    ids = torch.randint(-1, 999, (6, n), device=DEV, dtype=torch.int32)
    check(_ops().token_logprobs(x, ids, top_k=2), reference(x, ids, 2))


def test_strides_and_empty():
    ops = _ops()
    x, ids = make(4, 640, torch.bfloat16, 5)
    row = x[:1].expand(4, 640)  # one row, stride 0
    check(ops.token_logprobs(row, ids, top_k=3), reference(row, ids, 3))
    skip = make(8, 640, torch.float32, 6)[0][::2]
    check(ops.token_logprobs(skip, ids, top_k=3), reference(skip, ids, 3))
    n = ops.launch_count()
    out = ops.token_logprobs(x[:0], ids[:0], top_k=4)
    assert [tuple(a.shape) for a in out] == [(0,), (0,), (0, 4), (0, 4)] and ops.launch_count() == n


def test_confident_rows_keep_small_entropies():
    """Entropy and log p of rows with p near 1 are relative to their own size: ln S = log1p of
    what the other tokens weigh."""
    V = 4096
    gap = torch.tensor([4.0, 8.0, 12.0, 16.0], device=DEV)
    x = torch.full((4, V), -INF, device=DEV)
    x[:, 100] = 0.0
    x[:, 3000] = -gap
    ids = torch.full((4,), 100, device=DEV, dtype=torch.int32)
    out = _ops().token_logprobs(x, ids, top_k=3)
    ref = reference(x, ids, 3)
    # both tokens may fall to one thread's running fp32 sum: 2^-24 of 1 + e^-gap at most
    torch.testing.assert_close(out.logprobs.double().cpu(), ref[0], rtol=2**-19, atol=2**-23)
    torch.testing.assert_close(out.entropy.double().cpu(), ref[1], rtol=2**-18, atol=2**-22)
    assert torch.equal(out.top_ids.cpu().long(), ref[3])


def test_offsets_past_32_bits():
    """The last rows of logits of more than 2^32 bytes and 2^31 elements."""
    V, T = 163840, 13200
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=DEV)
    tail, ids = make(3, V, torch.bfloat16, 9)
    x[-3:] = tail
    all_ids = torch.zeros(T, dtype=torch.int32, device=DEV)
    all_ids[-3:] = ids
    out = _ops().token_logprobs(x, all_ids, top_k=4)
    check([a[-3:] for a in out], reference(tail, ids, 4))


def test_graph_and_streams():
    """Captured and replayed on new inputs, beside a call on another stream."""
    ops = _ops()
    x, ids = make(17, 30011, torch.bfloat16, 1)
    y, jds = make(17, 30011, torch.bfloat16, 2)
    a, b = x.clone(), ids.clone()
    ops.token_logprobs(a, b, top_k=6)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        out = ops.token_logprobs(a, b, top_k=6)
    torch.cuda.current_stream().wait_stream(s)
    for u, v in ((x, ids), (y, jds)):
        a.copy_(u)
        b.copy_(v)
        torch.cuda.synchronize()
        g.replay()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = ops.token_logprobs(y, jds, top_k=6)
        torch.cuda.synchronize()
        check(out, reference(u, v, 6))
        check(other, reference(y, jds, 6))


# ------------------------------------------------------------------ straight from hidden states
@pytest.mark.parametrize("T,V,K", [(1, 1, 8), (1, 300, 64), (7, 257, 72), (61, 10007, 1000), (128, 512, 256),
                                   (130, 2049, 520), (300, 1000, 2048), (1025, 5003, 136), (64, 102400, 256)])
def test_linear(T, V, K):
    """Products of bf16 are exact in fp32; a tensor-core sum of K of them is within K 2^-24 of
    the sum of their sizes (<= |x| |w|, Cauchy) whatever its order, or within 4 K 2^-24 should
    each step cut off instead of rounding, and log p of two logits moves by twice that."""
    ops = _ops()
    g = torch.Generator(device=DEV).manual_seed(T + V + K)
    x = torch.randn(T, K, device=DEV, generator=g).bfloat16()
    w = (torch.randn(V, K, device=DEV, generator=g) * (2.5 / math.sqrt(K))).bfloat16()
    ids = torch.randint(0, V, (T,), device=DEV, generator=g).int()
    ids[T // 2] = -1
    lp, ent = ops.linear_logprobs(x, w, ids)
    ref = reference(x.double() @ w.double().t(), ids, 0)
    size = float(x.double().norm(dim=1).max() * w.double().norm(dim=1).max())
    tol = 2 * 4 * K * 2**-24 * size + 2**-18
    torch.testing.assert_close(lp.double().cpu(), ref[0], rtol=2**-22, atol=tol)
    torch.testing.assert_close(ent.double().cpu(), ref[1], rtol=2**-18, atol=8 * tol)
    assert ops.status_word() == 0


@pytest.mark.parametrize("T,V,K", [(1, 20001, 200), (16, 50001, 72), (17, 50049, 136), (100, 60000, 328), (129, 64, 64),
                                   (200, 9000, 1104), (257, 130, 3000), (300, 50000, 200), (520, 700, 7168)])
def test_linear_shares(T, V, K):
    """Shares of one to seven units in tiles of unequal widths, on single CTAs and pairs; pairs
    whose second half has no rows or no tokens; segments that end inside K."""
    test_linear(T, V, K)


def test_linear_strides_and_empty():
    ops = _ops()
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn(40, 512, device=DEV, generator=g).bfloat16()
    w = torch.randn(700, 512, device=DEV, generator=g).bfloat16() * 0.1
    ids = torch.randint(0, 700, (20,), device=DEV, generator=g).int()
    x, v = big[::2, :256], w[:, 256:]
    lp, ent = ops.linear_logprobs(x, v, ids)
    same, same_ent = ops.linear_logprobs(x.contiguous(), v.contiguous(), ids)
    assert torch.equal(lp, same) and torch.equal(ent, same_ent)
    lp, ent = ops.linear_logprobs(x[:0], v, ids[:0])
    assert lp.shape == (0,) and ent.shape == (0,)


def test_linear_extreme_weights():
    """Logits up to 2e4 apart, equal logits, and a weight row with NaN."""
    ops = _ops()
    T, V, K = 33, 1030, 64
    g = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randint(-4, 5, (T, K), device=DEV, generator=g).bfloat16()
    w = torch.randint(-64, 65, (V, K), device=DEV, generator=g).bfloat16()  # whole numbers: exact logits
    w[5:9] = w[4]
    ids = torch.randint(0, V, (T,), device=DEV, generator=g).int()
    ids[3] = 7
    x[10] = 0
    lp, ent = ops.linear_logprobs(x, w, ids)
    ref = reference(x.double() @ w.double().t(), ids, 0)
    torch.testing.assert_close(lp.double().cpu(), ref[0], rtol=2**-22, atol=2**-18)
    torch.testing.assert_close(ent.double().cpu(), ref[1], rtol=2**-18, atol=2**-15)
    w[400, 3] = math.nan
    lp, ent = ops.linear_logprobs(x, w, ids)
    keep = (ids == -1).cpu()
    assert bool(torch.isnan(lp).cpu()[~keep].all()) and bool(torch.isnan(ent).all())
