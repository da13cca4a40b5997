"""Windowed attention on the GPU at the ends of its inputs: no kv rows, no requests, grids past a dimension's
limit, scores far from zero."""
import pytest
import torch

import plain_window as plain
from test_gpu_window import pool, prefill_reference, rows, run_prefill

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import vllm_paged_compression_amd as pkg
    import vllm_paged_compression_amd.ops as ops
    pkg.load_library()
    return ops


def cu(*sums):
    return torch.tensor(sums, dtype=torch.int32).cuda()


# ------------------------------------------------------------------ no kv rows
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 0), (20, 3)])
def test_prefill_without_kv_rows(ops, D, window, sinks):
    """No request has a kv row: zeros for their queries, the rows behind the last request left as they were."""
    g = torch.Generator().manual_seed(1)
    q = rows(g, 80, 4, D, torch.bfloat16).cuda()
    none = torch.empty(0, 2, D, dtype=torch.bfloat16, device="cuda")
    out = torch.full((80, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.prefill_window(q, none, none, cu(0, 1, 70), cu(0, 0, 0), 69, 0.1, window, sinks, out)
    assert got is out and (out[:70] == 0).all()
    assert (out[70:] == 7).all(), "rows behind the last request were touched"
    # (prefix sums that name rows which are not there are cut)
    out.fill_(7)
    ops.prefill_window(q, none, none, cu(0, 1, 70), cu(0, 5, 300), 69, 0.1, window, sinks, out)
    assert (out[:70] == 0).all() and (out[70:] == 7).all()


def test_prefill_without_kv_rows_refuses_what_the_call_refuses(ops):
    q = torch.zeros(3, 4, 72, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, 2, 72, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="head size"):
        ops.prefill_window(q, none, none, cu(0, 3), cu(0, 0), 3, 0.1, 5)


# ------------------------------------------------------------------ nothing to launch
@pytest.mark.parametrize("what", ["no requests", "max_q_len 0"])
def test_prefill_that_launches_nothing_returns_zeros(ops, what):
    """A fresh output is not left with what its memory held."""
    q, k = (torch.ones(50, h, 64, dtype=torch.float16, device="cuda") for h in (4, 2))
    for _ in range(4):
        dirty = torch.full((50, 4, 64), float("nan"), dtype=torch.float16, device="cuda")
        del dirty                                      # the allocator hands the same memory out again
        sums = cu(0) if what == "no requests" else cu(0, 0)
        got = ops.prefill_window(q, k, k, sums, sums, 0, 0.1, 5)
        assert got.shape == q.shape and (got == 0).all()
    out = torch.full((50, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    ops.prefill_window(q, k, k, sums, sums, 0, 0.1, 5, 0, out)
    assert (out == 7).all()                            # a caller's output keeps the rows of no request


# ------------------------------------------------------------------ grids
@pytest.mark.parametrize("Hq,H,D", [(4, 1, 64), (4, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("max_q_len", [16 * 65535, 16 * 65535 + 1, 64 * 65535])
def test_prefill_max_q_len_far_above_the_prompts(ops, Hq, H, D, max_q_len):
    """max_q_len sizes the grid: with the query heads of a KV head side by side a workgroup takes 16 rows, which
    more than 65535 workgroups in a row would have to cover."""
    g = torch.Generator().manual_seed(2)
    lens = [100, 31]
    q, k, v = (rows(g, 131, h, D, torch.bfloat16) for h in (Hq, H, H))
    got = ops.prefill_window(q.cuda(), k.cuda(), v.cuda(), cu(0, 100, 131), cu(0, 100, 131), max_q_len, D ** -0.5, 17, 2)
    plain.assert_within(got, *prefill_reference(q, k, v, lens, lens, 17, 2, D ** -0.5))


# ------------------------------------------------------------------ scores far from zero
def far_scores(dtype, D, size, sign, n, ahead):
    """q, k with every score sign * size but one key's, which is ahead by half of it; D ** -0.5 scales."""
    per = (size / D ** 0.5) ** 0.5
    q = torch.full((n, 2, D), sign * per).to(dtype)
    k = torch.full((n, 1, D), per).to(dtype)
    k[ahead] *= 1.5 if sign > 0 else 0.5
    return q, k


SIZES = [(torch.float16, s) for s in (1e4, 1e8, 1e9, 1e10)] + [(torch.bfloat16, s) for s in (1e4, 1e9, 1e10, 1e25, 1e33)]


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_decode_window_scores_far_from_zero(ops, dtype, size, sign):
    g = torch.Generator().manual_seed(4)
    D, bs, n, ahead = 64, 16, 200, 77
    kc, vc, t = pool(g, [n], 1, D, bs, dtype)
    q, k = far_scores(dtype, D, size, sign, n, ahead)
    for j in range(n):
        kc[t[0, j // bs].long(), :, :, j % bs] = k[j].view(1, D // 8, 8)
    want = vc[t[0, ahead // bs].long(), 0, :, ahead % bs]
    ln = torch.tensor([n], dtype=torch.int32)
    for max_len in (64, n, 1 << 16):
        out = torch.empty_like(q[:1]).cuda()
        ops.paged_attention_window(out, q[:1].cuda(), kc.cuda(), vc.cuda(), 1, D ** -0.5, t.cuda(), ln.cuda(), bs,
                                   max_len, 150, 2)
        assert torch.equal(out.cpu(), want.expand(1, 2, D)), f"launch shaped for {max_len} tokens"
