"""Log probabilities in the serving loop, prompt scoring, and several answers to one prompt
that share cache pages."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg():
    from sparkpipe_rs_b200.models.config import v2_lite

    return v2_lite().replace(name="small-mla-moe", num_layers=3, hidden_size=1024, n_routed_experts=16,
                             num_experts_per_tok=4, moe_intermediate_size=256, intermediate_size=2048,
                             n_shared_experts=1, vocab_size=4096, first_k_dense_replace=1, init_std=0.05)


@pytest.fixture(scope="module")
def model():
    from sparkpipe_rs_b200.models.mla_moe import MLAMoEModel

    return MLAMoEModel(_cfg(), seed=0, device="cuda", max_positions=1024)


def _engine(model, **kw):
    from sparkpipe_rs_b200.serving.engine import EngineConfig, LLMEngine

    kw = {"max_batch": 4, "block_size": 64, "max_model_len": 512, "max_prefill_tokens": 256,
          "decode_buckets": (1, 2, 4), **kw}
    return LLMEngine(model.cfg, EngineConfig(**kw), model=model, device="cuda")


def _prompts():
    g = torch.Generator().manual_seed(0)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (40, 65, 300, 9)]


@pytest.mark.parametrize("kw", [{}, {"async_decode": False}, {"use_cuda_graph": False}, {"kv_cache_dtype": "fp8"}])
def test_engine_logprobs(model, kw):
    """The same tokens as without log probabilities (a 300-token prompt in two chunks among
    them); a greedy token is the first alternative, a sampled one need not be."""
    from sparkpipe_rs_b200.serving.engine import SamplingParams

    plain, scored = _engine(model, **kw), _engine(model, logprobs=3, **kw)
    for params in (SamplingParams(max_tokens=9, ignore_eos=True),
                   SamplingParams(max_tokens=7, temperature=1.5, seed=3, ignore_eos=True)):
        a, b = plain.generate(_prompts(), params).outputs, scored.generate(_prompts(), params).outputs
        assert [o.token_ids for o in a] == [o.token_ids for o in b]
        assert not a[0].logprobs
        for o in b:
            assert len(o.logprobs) == len(o.entropies) == len(o.top_logprobs) == len(o.token_ids)
            for tok, lp, ent, top in zip(o.token_ids, o.logprobs, o.entropies, o.top_logprobs):
                assert len(top) == 3 and top[0][1] >= top[1][1] >= top[2][1] >= -math.log(4096) * 4
                assert 0.0 < ent <= math.log(4096) + 1e-4 and lp <= top[0][1]
                if params.temperature == 0:
                    assert (tok, lp) == top[0]
    assert _engine(model, logprobs=0).generate(_prompts()[:1], SamplingParams(max_tokens=2)).outputs[0].top_logprobs == [[], []]


def test_engine_logprobs_refused(model):
    with pytest.raises(ValueError, match="speculation"):
        _engine(model, logprobs=2, speculation="chain")
    with pytest.raises(ValueError, match="at most 32"):
        _engine(model, logprobs=33)


def test_score(model):
    """Prompt scores against the log softmax of the model's own bf16 logits: each logit is
    rounded by at most 2^-8 of its size (finfo.eps / 2), so a log probability, a difference of
    two of them, moves by at most 2^-7 of the largest logit; 2^-12 covers the fp32 sums."""
    from sparkpipe_rs_b200.models.mla_moe import ForwardBatch

    eng = _engine(model)
    prompts = [[5], *_prompts()[:2], [7, 7], _prompts()[3], _prompts()[2][:256]]
    got = eng.score(prompts)
    assert [len(g) for g in got] == [len(p) - 1 for p in prompts]
    for p, g in zip(prompts, got):
        T = len(p)
        i32 = dict(dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, T], **i32)
        fb = ForwardBatch(mode="prefill", token_ids=torch.tensor(p, **i32), positions=torch.arange(T, **i32),
                          slot_mapping=torch.full((T,), -1, **i32), cu_q=cu, cu_k=cu, max_q=T)
        logits = model.forward(fb, eng.cache).double()
        want = torch.log_softmax(logits, 1)[:-1].gather(1, torch.tensor(p[1:], device="cuda").view(-1, 1))[:, 0]
        tol = 2**-7 * float(logits.abs().max()) + 2**-12
        torch.testing.assert_close(torch.tensor(g, dtype=torch.float64), want.cpu(), rtol=0, atol=tol)
    assert eng.score([]) == [] and eng.score([[1]]) == [[]]
    for bad in ([1] * 257, [4096, 1], [-1, 2]):
        with pytest.raises(ValueError, match="score"):
            eng.score([bad])


def _answers(model, n, kv_dtype="bf16", blocks=40, top=2):
    from sparkpipe_rs_b200.models.mla_moe import KVCache
    from sparkpipe_rs_b200.serving.answers import ParallelAnswers

    cache = KVCache(model.cfg, num_blocks=blocks, block_size=64, device="cuda", kv_dtype=kv_dtype)
    return ParallelAnswers(model, cache, n, 320, top_logprobs=top), cache


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("plen", [1, 63, 64, 100])
def test_answers_share_the_prompt(model, kv_dtype, plen, monkeypatch):
    """Answers whose pages are shared and copied on their first write equal answers that had
    whole copies of the prompt's pages from the start, token for token, and so does every score."""
    from sparkpipe_rs_b200 import ops

    prompt = _prompts()[2][:plen]
    pa, _ = _answers(model, 4, kv_dtype)
    got = pa.generate(prompt, 70, temperature=1.0, seed=5, keep=4)
    assert len({tuple(a.token_ids) for a in got}) == 4  # four draws
    assert [a.mean_logprob for a in got] == sorted((a.mean_logprob for a in got), reverse=True)
    apart, cache = _answers(model, 4, kv_dtype, blocks=48)

    def four_rows(table, lens, parents, refs, block_size=64):
        rows, pages = [table[0]], -(-plen // 64)
        for _ in range(3):
            row = torch.full_like(table, -1)
            short = ops.reserve_pages(row, torch.zeros_like(lens), refs, cache.data, lens, cache_scales=cache.scales)
            assert int(short.sum()) == 0
            ops.copy_pages(cache.data, table[0, :pages].contiguous(), row[0, :pages].contiguous(),
                           cache_scales=cache.scales)
            rows.append(row[0])
        return torch.stack(rows).contiguous(), lens.expand(4).contiguous()

    with monkeypatch.context() as mp:
        mp.setattr(ops, "fork_pages", four_rows)
        want = apart.generate(prompt, 70, temperature=1.0, seed=5, keep=4)
    for a, b in zip(got, want):
        assert a.token_ids == b.token_ids and a.logprobs == b.logprobs and a.entropies == b.entropies
        assert a.top_logprobs == b.top_logprobs and len(a.token_ids) == 70
    # pages: the prompt's whole ones once, the rest per answer, all at the front of the cache
    whole = plen // 64
    per = -(-(plen + 69) // 64) - whole
    used = whole + 4 * per
    refs = pa.refs.cpu()
    assert int((refs > 0).sum()) == used and bool((refs[:used] > 0).all())
    assert sorted(refs[:used].tolist()) == [1] * (4 * per) + [4] * whole
    assert ops.status_word() == 0


def test_answers_keep_and_stop(model):
    """Losers give their pages back; stop tokens end an answer; equal seeds repeat; greedy answers agree."""
    pa, cache = _answers(model, 5)
    prompt = _prompts()[1]
    a = pa.generate(prompt, 30, seed=1, keep=2)
    assert len(a) == 2 and pa.table.shape[0] == 2 and pa.lens.tolist() == [len(prompt) + 29] * 2
    assert int((pa.refs > 0).sum()) == len(prompt) // 64 + 2 * (-(-(len(prompt) + 29) // 64) - len(prompt) // 64)
    b = pa.generate(prompt, 30, seed=1, keep=5)
    assert [x.token_ids for x in b[:2]] == [x.token_ids for x in a]
    stop = b[0].token_ids[7]
    c = pa.generate(prompt, 30, seed=1, keep=5, stop_token_ids=(stop,))
    for x in c:
        assert stop not in x.token_ids[:-1] and (x.token_ids[-1] == stop or len(x.token_ids) == 30)
        assert any(x.token_ids == y.token_ids[:len(x.token_ids)] and x.logprobs == y.logprobs[:len(x.logprobs)] for y in b)
    g = pa.generate(prompt, 12, temperature=0.0, keep=5)
    assert len({tuple(x.token_ids) for x in g}) == 1 and len({tuple(x.logprobs) for x in g}) == 1
    assert all(t == top[0][0] for t, top in zip(g[0].token_ids, g[0].top_logprobs))


def test_answers_refused(model):
    pa, _ = _answers(model, 2, blocks=3)
    for args in (([], 4), ([1], 0), ([1] * 300, 30), ([4096], 4), ([-1], 4)):
        with pytest.raises(ValueError):
            pa.generate(*args)
    with pytest.raises(ValueError, match="positions"):
        type(pa)(model, pa.cache, 2, 1025)
    with pytest.raises(ValueError, match="keep"):
        pa.generate([1, 2], 3, keep=3)
    with pytest.raises(MemoryError, match="prompt"):
        pa.generate([1] * 200, 3)
    with pytest.raises(MemoryError, match="ran out"):
        pa.generate([1] * 100, 60)  # two pages of prompt, a copy of the second, and no third for both
    assert len(pa.generate([1] * 60, 3, keep=2)) == 2


def test_answers_out_of_pages(model, monkeypatch):
    """Too few pages end a call before its first step, or with stop tokens soon after the page is missing, and
    not at the end of the answers; the next call starts afresh."""
    pa, _ = _answers(model, 2, blocks=3)
    steps = []
    run = pa.graph.run
    monkeypatch.setattr(pa.graph, "run", lambda: (steps.append(1), run())[1])
    with pytest.raises(MemoryError, match="ran out"):
        pa.generate([1] * 100, 200)
    assert not steps
    with pytest.raises(MemoryError, match="ran out"):
        pa.generate([1] * 100, 200, stop_token_ids=(-2,))
    assert 28 <= len(steps) <= 30  # tokens 100 to 127 fit, the third page of both rows does not
    for plen, new, fits in ((100, 29, True), (100, 30, False), (64, 65, True), (64, 66, False), (128, 1, True)):
        if fits:
            assert [len(a.token_ids) for a in pa.generate([1] * plen, new, keep=2)] == [new, new]
            continue
        with pytest.raises(MemoryError, match="ran out"):
            pa.generate([1] * plen, new, keep=2)
    for top in (-1, 33):
        with pytest.raises(ValueError, match="alternatives"):
            type(pa)(model, pa.cache, 2, 320, top_logprobs=top)
