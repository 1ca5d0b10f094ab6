"""Arguments that the log-probability and page operators refuse, on any machine: shapes, types
and strides are checked before the device, and CPU tensors never reach a kernel."""
import pytest
import torch


def _ops():
    from sparkpipe_rs_b200 import ops

    return ops


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("logits,ids,k,says", [
    (torch.zeros(4, 40), i32(4), 33, "top_k"),
    (torch.zeros(4, 9), i32(4), 10, "top_k"),
    (torch.zeros(4, 9), i32(4), -1, "top_k"),
    (torch.zeros(4, 0), i32(4), 0, "no columns"),
    (torch.zeros(9, 4).t(), i32(4), 1, "unit column stride"),
    (torch.zeros(36), i32(36), 1, "unit column stride|out of range|Dimension"),
    (torch.zeros(4, 9, dtype=torch.float64), i32(4), 1, "bf16, fp16 or fp32"),
    (torch.zeros(4, 9), i32(3), 1, "one row per logits row"),
    (torch.zeros(4, 9), i32(4, 2, 2), 1, "one row per logits row"),
    (torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64), 1, "int32"),
    (torch.zeros(4, 9), i32(4, 6)[:, ::2], 1, "contiguous"),
    (torch.zeros(4, 9), i32(4), 1, "CUDA"),
])
def test_token_logprobs(logits, ids, k, says):
    with pytest.raises((ValueError, RuntimeError), match=says):
        _ops().token_logprobs(logits, ids, top_k=k)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("x,w,ids,says", [
    (_bf(4, 16), _bf(9, 16), i32(3), "one per row"),
    (_bf(4, 16), _bf(9, 16), i32(4, 1), "one per row"),
    (_bf(4, 12), _bf(9, 12), i32(4), "multiple of 8"),
    (_bf(4, 16), _bf(9, 24), i32(4), "x .T, K. and w"),
    (_bf(4, 16), _bf(0, 16), i32(4), "no columns"),
    (_bf(4, 16).float(), _bf(9, 16), i32(4), "bf16"),
    (_bf(4, 16), _bf(9, 16), torch.zeros(4, dtype=torch.int64), "int32"),
    (_bf(4, 20)[:, :16], _bf(9, 16), i32(4), "16-byte aligned"),
    (_bf(4, 24)[:, 1:17], _bf(9, 16), i32(4), "16-byte aligned"),
    (_bf(1, 16).expand(4, 16), _bf(9, 16), i32(4), "16-byte aligned"),
    (_bf(16, 4).t(), _bf(9, 16), i32(4), "row-major"),
    (_bf(4, 16), _bf(9, 16), i32(4), "CUDA"),
])
def test_linear_logprobs(x, w, ids, says):
    with pytest.raises((ValueError, RuntimeError), match=says):
        _ops().linear_logprobs(x, w, ids)


CACHE = _bf(2, 128, 8)


@pytest.mark.parametrize("data,scales,src,dst,bs,says", [
    (_bf(2, 128), None, i32(2), i32(2), 64, "layers, slots, row"),
    (_bf(2, 100, 8), None, i32(2), i32(2), 64, "whole pages"),
    (_bf(2, 128, 8), None, i32(2), i32(2), 0, "whole pages"),
    (_bf(2, 128, 9), None, i32(2), i32(2), 64, "4-byte words"),
    (_bf(2, 128, 16)[:, :, :8], None, i32(2), i32(2), 64, "dense slots"),
    (_bf(1, 128, 8).expand(2, 128, 8), None, i32(2), i32(2), 64, "overlap"),
    (CACHE, torch.zeros(2, 64, 5), i32(2), i32(2), 64, "layers and slots"),
    (CACHE, None, i32(3), i32(2), 64, "source for every destination"),
    (CACHE, None, torch.zeros(2), i32(2), 64, "int32"),
    (CACHE, None, i32(2), i32(2), 64, "CUDA"),
])
def test_copy_pages(data, scales, src, dst, bs, says):
    with pytest.raises((ValueError, RuntimeError), match=says):
        _ops().copy_pages(data, src, dst, block_size=bs, cache_scales=scales)


@pytest.mark.parametrize("table,lens,parents,refs,bs,says", [
    (i32(3, 4), i32(3), i32(2), torch.zeros(9), 64, "refs"),
    (i32(3, 4), i32(3), i32(2), i32(0), 64, "refs"),
    (i32(3, 4).t(), i32(4), i32(2), i32(9), 64, "block_table"),
    (i32(3, 4), i32(2), i32(2), i32(9), 64, "one length"),
    (i32(3, 4), i32(3), torch.zeros(2, dtype=torch.int64), i32(9), 64, "int32"),
    (i32(3, 4), i32(3), i32(2), i32(9), 0, "block_size"),
    (i32(3, 4), i32(3), i32(2), i32(9), 64, "CUDA"),
])
def test_fork_pages(table, lens, parents, refs, bs, says):
    with pytest.raises((ValueError, RuntimeError), match=says):
        _ops().fork_pages(table, lens, parents, refs, block_size=bs)


@pytest.mark.parametrize("table,lens,refs,tokens,says", [
    (i32(3, 4), i32(2), i32(2), 1, "one length"),
    (i32(3, 4), i32(3), i32(3), 1, "more pages than the cache"),
    (i32(3, 4), i32(3), i32(2), -1, "negative"),
    (i32(3, 4), i32(3), i32(2), i32(2), "token count"),
    (i32(1025, 1), i32(1025), i32(2), 1, "at most 1024 rows"),
    (i32(3, 4), i32(3), i32(2), 1, "CUDA"),
])
def test_reserve_pages(table, lens, refs, tokens, says):
    with pytest.raises((ValueError, RuntimeError), match=says):
        _ops().reserve_pages(table, lens, refs, CACHE, tokens)


def test_free_and_compact():
    ops = _ops()
    for rows, says in ((i32(2, 2), "rows must be"), (torch.zeros(2), "int32"), (i32(2), "CUDA"), (None, "CUDA")):
        with pytest.raises((ValueError, RuntimeError), match=says):
            ops.free_pages(i32(3, 4), i32(2), rows)
    assert ops.kernels().LOGPROBS_MAX_TOP == 32 and ops.kernels().PAGES_MAX_ROWS == 1024
    for refs, says in ((i32(3), "more pages than the cache"), (i32(2), "CUDA")):
        with pytest.raises((ValueError, RuntimeError), match=says):
            ops.compact_pages(i32(3, 4), refs, CACHE)


def test_too_many_pieces():
    """Caches of more pieces than one call counts are refused before an index kernel changes tables or counts."""
    ops = _ops()
    n = 1 << 20
    data = torch.empty(2048, n, 4, dtype=torch.uint8, device="meta")  # 2,048 layers of a million 4-byte pages
    with pytest.raises(RuntimeError, match="compact_pages: too many pieces"):
        ops.compact_pages(i32(3, 4), i32(n), data, block_size=1)
    with pytest.raises(RuntimeError, match="copy_pages: too many pieces"):
        ops.copy_pages(data, i32(n // 2), i32(n // 2), block_size=1)
    wide = torch.empty(1 << 20, 1024, 16, dtype=torch.uint8, device="meta")  # a million layers of 1,024 pages
    with pytest.raises(RuntimeError, match="reserve_pages: too many pieces"):
        ops.reserve_pages(i32(1024, 4), i32(1024), i32(1024), wide, block_size=1)
    for few in (data[:2047], wide[:, :1023]):  # one layer, or one page, less
        with pytest.raises(RuntimeError, match="CUDA"):
            ops.copy_pages(few, i32(n // 2), i32(n // 2), block_size=1)


def test_engine_config_order():
    """A setting that came later stands last: those before it keep their places."""
    from dataclasses import fields

    from sparkpipe_rs_b200.serving.engine import EngineConfig

    names = [f.name for f in fields(EngineConfig)]
    assert names[-1] == "logprobs" and names[names.index("warm_prefill") + 1] == "prefill_graphs"
