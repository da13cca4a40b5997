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
    for _ in range(4):                                 # a fresh output is all zeros, whatever its memory held
        dirty = torch.full_like(out, float("nan"))
        del dirty
        assert (ops.prefill_window(q, none, none, cu(0, 1, 70), cu(0, 0, 0), 69, 0.1, window, sinks) == 0).all()
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


# ------------------------------------------------------------------ prefill scores far from zero
@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [100, 300])
def test_prefill_scores_far_from_zero(ops, dtype, size, sign, D, window):
    """Rows that see one key far ahead of the others return its value; rows before it see equal scores and return
    the mean of their values."""
    g = torch.Generator().manual_seed(3)
    n, ahead = 500, 150
    q, k = far_scores(dtype, D, size, sign, n, ahead)
    v = rows(g, n, 1, D, dtype)
    # (one request takes the shape of launches that leave compute units idle, 40 take those of large ones)
    for copies in (1, 40):
        lens = [n] * copies
        got = run_prefill(ops, *(x.repeat(copies, 1, 1) for x in (q, k, v)), lens, lens, window, 0, D ** -0.5).cpu()
        for c in range(0, copies, 13):
            one = got[c * n:(c + 1) * n]
            assert torch.equal(one[ahead:ahead + window], v[ahead].expand(window, 2, D)), f"request {c} of {copies}"
            mean = torch.stack([v[max(0, i - window + 1):i + 1].double().mean(0) for i in range(ahead)])
            spread = torch.stack([v[max(0, i - window + 1):i + 1].double().abs().mean(0) for i in range(ahead)])
            # equal weights: one rounding of the mean, and f32 sums of up to 100 products
            u = plain.HALF_STEP[dtype]
            plain.assert_within(one[:ahead], mean.expand(ahead, 2, D),
                                (mean.abs() * u + spread * (200 * 2.0 ** -24)
                                 + 2.0 ** -25 * (dtype == torch.float16)).expand(ahead, 2, D), f"request {c} of {copies}")


@pytest.mark.parametrize("dtype,big", [(torch.float16, 6e4), (torch.bfloat16, 1e5), (torch.bfloat16, 1e12)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(100, 0), (300, 5), (0, 0)])
def test_prefill_scores_near_and_far_from_zero(ops, dtype, big, D, window, sinks):
    """Keys far below the others (the first tile, every seventh key after it) and one far above: far keys have no
    weight beside near ones, a row that sees far ones alone returns their mean."""
    g = torch.Generator().manual_seed(5)
    n, above = 420, 350
    i = torch.arange(n)
    low = (i < 70) | (i % 7 == 0)
    q, k, v = rows(g, n, 2, D, dtype), rows(g, n, 1, D, dtype), rows(g, n, 1, D, dtype)
    q[:, :, 0], k[:, :, 0] = big, 0.0
    k[low] = 0.0
    k[low, :, 0] = -big
    k[above, :, 0] = big
    see = i[None] <= i[:, None]
    if window:
        see &= (i[None] > i[:, None] - window) | (i[None] < sinks)
    heaviest = torch.where(i == above, 2, torch.where(low, 0, 1))[None].expand(n, n).masked_fill(~see, -1)
    see &= heaviest == heaviest.amax(1, keepdim=True)
    # near keys: attend_one's terms with prefill_reference's two (both in 64 bits, over the keys that count)
    qn, kn = q.double().clone(), k.double().clone()
    qn[:, :, 0] = 0                                     # what the keys that count together differ by
    s = torch.matmul(qn.transpose(0, 1), kn[:, 0].T.contiguous()) * D ** -0.5
    size = (torch.matmul(qn.abs().transpose(0, 1), kn[:, 0].abs().T.contiguous()) * D ** -0.5 * see).amax(2, keepdim=True)
    p = torch.softmax(s.masked_fill(~see, float("-inf")), 2)
    vv, u = v[:, 0].double(), plain.HALF_STEP[dtype]
    ref, spread = torch.matmul(p, vv).transpose(0, 1), torch.matmul(p, vv.abs())
    rel = 2 * u + 2 * size * (D + 4) * 2.0 ** -24 + 4 * 2.0 ** -22 + 2 * n * 2.0 ** -24
    bound = (spread * rel).transpose(0, 1) + ref.abs() * u
    heavy = torch.matmul(see.double(), vv.abs())[:, None] / torch.exp(s.masked_fill(~see, float("-inf"))
                                                                     - s.masked_fill(~see, float("-inf")).amax(2, keepdim=True)).sum(2).T[..., None]
    bound = bound + heavy * (2.0 ** -120 if dtype == torch.bfloat16 else 2.0 ** -19) + 2.0 ** -25 * (dtype == torch.float16)
    for copies in (1, 40):
        lens = [n] * copies
        got = run_prefill(ops, *(x.repeat(copies, 1, 1) for x in (q, k, v)), lens, lens, window, sinks, D ** -0.5).cpu()
        for c in range(0, copies, 13):
            plain.assert_within(got[c * n:(c + 1) * n], ref, bound, f"request {c} of {copies}")


# ------------------------------------------------------------------ memory
def test_out_of_memory_is_torchs_error(ops):
    """A fresh output that the allocator refuses: the exception that servers catch, and the next call works."""
    q, k = (torch.ones(1 << 16, h, 128, dtype=torch.float16, device="cuda") for h in (4, 1))
    sums = cu(0, 40)
    torch.cuda.empty_cache()
    held = []
    try:
        torch.cuda.set_per_process_memory_fraction(1e-4)
        with pytest.raises(torch.cuda.OutOfMemoryError):    # what other tests' tensors leave free of their segments
            while True:
                held.append(torch.empty(1 << 25, dtype=torch.uint8, device="cuda"))
        with pytest.raises(torch.cuda.OutOfMemoryError):
            ops.prefill_window(q, k, k, sums, sums, 40, 0.1, 5)
    finally:
        del held
        torch.cuda.set_per_process_memory_fraction(1.0)
    out = ops.prefill_window(q, k, k, sums, sums, 40, 0.1, 5)
    assert (out[:40] == 1).all()
