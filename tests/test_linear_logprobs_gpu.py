"""linear_logprobs in each of its forms: CTA pairs and single CTAs, accumulators of 256, 512 and 1,024 of K, ring stages
of one and two K blocks, on problems of several segments and ragged ends."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"

# (T, V, K) and (CTAs of a tile, K blocks of 64 in a segment, K blocks of a stage) on 148 SMs
FORMS = [
    (1, 30045, 1160, (1, 4, 1)), (61, 102397, 1032, (1, 4, 1)), (128, 90001, 520, (1, 4, 1)),
    (3, 1500, 2056, (1, 4, 2)), (61, 10007, 1000, (1, 4, 2)), (128, 700, 7168, (1, 4, 2)),
    (300, 50000, 2056, (1, 8, 1)), (313, 9534, 1104, (1, 8, 1)),
    (1025, 5003, 1096, (2, 8, 1)), (2000, 9001, 2056, (2, 8, 1)), (1000, 32767, 1544, (2, 8, 1)),
    (200, 9000, 1104, (2, 8, 2)), (520, 700, 7168, (2, 8, 2)),
    (256, 102397, 1032, (2, 16, 1)), (150, 33000, 2056, (2, 16, 1)), (129, 32769, 3080, (2, 16, 1)),
    (1100, 40000, 1544, (2, 16, 1)),
]


def _ops():
    from sparkpipe_rs_b200 import ops

    return ops


def check_form(T, V, K, form):
    """The problem takes the form that the case is there for (where the card has as many SMs as it was chosen on)."""
    k = _ops().kernels()
    if k.num_sms() == 148:
        assert k.linear_logprobs_plan(T, V, K, 148)[:3] == form


def reference(logits, ids):
    """(logprobs, entropy) in 64 bits."""
    z = torch.log_softmax(logits.double(), 1)
    given = torch.where(ids < 0, 0.0, z.gather(1, ids.long().clamp(min=0)[:, None])[:, 0])
    return given, -(z.exp() * z).sum(1)


@pytest.mark.parametrize("T,V,K,form", FORMS)
def test_whole_numbers(T, V, K, form):
    """Whole-number operands: every partial sum is a whole number below 2^24, so the logits are exact in whatever
    order and segments they are added, and what is left are the sums of the softmax: log p within 2^-18 (one fp32
    rounding of |t| < 64 twice is 2^-18 / 2, ln S within 2^-19), entropy, a mean of |t|, within 2^-18 of itself and
    2^-15. A K block, half a tile or a share left out moves log p by whole numbers. All logits lie around 1,024,
    where bf16 holds every eighth number: rounded logits are far off."""
    ops = _ops()
    check_form(T, V, K, form)
    g = torch.Generator(device=DEV).manual_seed(T + V + K)
    x = torch.zeros(T, K, device=DEV)
    at = torch.randint(0, K, (T, 24), device=DEV, generator=g)
    x.scatter_(1, at, torch.randint(0, 2, (T, 24), device=DEV, generator=g) * 2.0 - 1.0)
    w = torch.randint(-1, 2, (V, K), device=DEV, generator=g).float()
    for k in (K // 5, K - 3):  # 512 each for every token
        x[:, k], w[:, k] = 16, 32
    x, w = x.bfloat16(), w.bfloat16()
    ids = torch.randint(0, V, (T,), device=DEV, generator=g).int()
    ids[0], ids[T // 2] = V - 1, -1 if T > 1 else V - 1
    lp, ent = ops.linear_logprobs(x, w, ids)
    logits = x.double() @ w.double().t()
    want, want_ent = reference(logits, ids)
    torch.testing.assert_close(lp.double(), want, rtol=2**-22, atol=2**-18)
    torch.testing.assert_close(ent.double(), want_ent, rtol=2**-18, atol=2**-15)
    rounded, rounded_ent = reference(logits.float().bfloat16(), ids)
    live = ids >= 0
    assert float((rounded - want)[live].abs().max()) > 2**-8 and float((rounded_ent - want_ent).abs().max()) > 2**-8
    assert ops.status_word() == 0


@pytest.mark.parametrize("T,V,K,form", FORMS)
def test_accuracy(T, V, K, form):
    """Random operands, 2-norms relative to 64 bits. An MMA adds 16 products to its accumulator and cuts the sum off
    below its last bit, on average by half a unit, 2^-24 of the accumulator at most; over the n = 4 x segment MMAs of a
    segment the accumulator grows like a random walk, 2/3 of its last size on average, so a logit shrinks by up to
    n (2/3) 2^-24 of itself, all logits the same way. With logits of variance 4 that moves the entropy (ln V - 2, at
    least 4.5 here) by 4 times and log p (around -ln V - 2) by some 4 times as much, less than it relative to themselves.
    2^-21 is for the sums of the softmax. Logits rounded to bf16 (off by up to 2^-8 of themselves, either way) fail."""
    ops = _ops()
    check_form(T, V, K, form)
    g = torch.Generator(device=DEV).manual_seed(T + V + K)
    x = torch.randn(T, K, device=DEV, generator=g).bfloat16()
    w = (torch.randn(V, K, device=DEV, generator=g) * (2.0 / K**0.5)).bfloat16()
    ids = torch.randint(0, V, (T,), device=DEV, generator=g).int()
    lp, ent = ops.linear_logprobs(x, w, ids)
    logits = x.double() @ w.double().t()
    want = reference(logits, ids)
    tol = form[1] * 4 * (2 / 3) * 2**-24 + 2**-21

    def off(got, ref):
        return float((got.double() - ref).norm() / ref.norm())

    assert off(lp, want[0]) < tol and off(ent, want[1]) < tol
    rounded = reference(logits.float().bfloat16(), ids)
    assert off(rounded[0], want[0]) > tol and off(rounded[1], want[1]) > tol


@pytest.mark.parametrize("T,shares", [(9472, 2), (18944, 1)])
def test_few_shares(T, shares):
    """So many row tiles that a thread's running sums take in 320 or all 640 tiles of a row, whose rounding errors they
    keep: first and last rows within 2^-21 for the terms (exp2's 2^-22, the product before it 2^-23) and the roundings
    at the end (2^-23 together)."""
    ops = _ops()
    V, K, n = 163840, 64, 192
    if ops.kernels().num_sms() == 148:
        assert ops.kernels().linear_logprobs_plan(T, V, K, 148)[4] == shares
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, K, device=DEV, generator=g).bfloat16()
    w = (torch.randn(V, K, device=DEV, generator=g) * 0.25).bfloat16()
    ids = torch.randint(0, V, (T,), device=DEV, generator=g).int()
    lp, ent = ops.linear_logprobs(x, w, ids)
    for rows in (slice(0, n), slice(T - n, T)):
        want, want_ent = reference(x[rows].double() @ w.double().t(), ids[rows])
        assert float((lp[rows].double() - want).norm() / want.norm()) < 2**-21
        assert float((ent[rows].double() - want_ent).norm() / want_ent.norm()) < 2**-21


@pytest.mark.parametrize("T,V,K", [(17, 5000, 200), (300, 9534, 1104), (200, 33000, 1032)])
def test_graph_and_streams(T, V, K):
    """Captured and replayed on new inputs, beside a call on another stream: each its own workspace, and the same
    bits as a call by itself. Two graphs replayed at the same time too."""
    ops = _ops()
    g = torch.Generator(device=DEV).manual_seed(V)

    def make():
        return (torch.randn(T, K, device=DEV, generator=g).bfloat16(),
                (torch.randn(V, K, device=DEV, generator=g) * (2.0 / K**0.5)).bfloat16(),
                torch.randint(0, V, (T,), device=DEV, generator=g).int())

    first, second = make(), make()
    want = [[a.clone() for a in ops.linear_logprobs(*p)] for p in (first, second)]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    held, outs, graphs = [], [], []
    for stream in (s, t):
        mine = [a.clone() for a in first]
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            out = ops.linear_logprobs(*mine)
        held.append(mine)
        outs.append(out)
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(4):
        order = (first, second) if turn % 2 == 0 else (second, first)
        for mine, new in zip(held, order):
            for a, b in zip(mine, new):
                a.copy_(b)
        torch.cuda.synchronize()
        for stream, graph in zip((s, t), graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        beside = ops.linear_logprobs(*second)
        torch.cuda.synchronize()
        for out, i in zip(outs, (0, 1) if turn % 2 == 0 else (1, 0)):
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
        assert torch.equal(beside[0], want[1][0]) and torch.equal(beside[1], want[1][1])
    assert ops.status_word() == 0


def test_entropy_of_one_long_share():
    """A thread's sums over all 640 tiles of a row, with the tiles' rounding errors kept: what is left is the rounding
    of a part's E (2^-24 of it, E / S being 0.55 of the entropy here), of ln S (0.46 of it) and of the entropy, 2^-23
    together, and with plain fp32 sums it was 2^-22.7."""
    ops = _ops()
    T, V, K, n = 18944, 163840, 64, 256
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(T, K, device=DEV, generator=g).bfloat16()
    w = (torch.randn(V, K, device=DEV, generator=g) * 0.3125).bfloat16()
    ids = torch.zeros(T, dtype=torch.int32, device=DEV)
    ent = ops.linear_logprobs(x, w, ids)[1]
    for rows in (slice(0, n), slice(T // 2, T // 2 + n), slice(T - n, T)):
        want = reference(x[rows].double() @ w.double().t(), ids[rows])[1]
        assert float((ent[rows].double() - want).norm() / want.norm()) < 2**-23
