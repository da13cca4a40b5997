"""Attention with a sliding window and sink tokens on the GPU: the prefill over dense rows and the decode
over a 16-bit paged cache, against a plain implementation in 64 bits."""
import pytest
import torch

import plain_window as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import vllm_paged_compression_amd as pkg
    import vllm_paged_compression_amd.ops as ops
    pkg.load_library()
    return ops


def rows(g, n, heads, D, dtype):
    return (torch.randn(n, heads, D, generator=g) * torch.exp(0.5 * torch.randn(heads, D, generator=g))).to(dtype)


def prefill_reference(q, k, v, q_lens, kv_lens, window, sinks, scale):
    """(out, bound) f64 [Tq, Hq, D], from the definition; see attend_one for the bound's terms.  Two more
    belong to this kernel: its sums are those of the rounded weights, so a rounding in them moves
    numerator and denominator alike and the u per weight stays; its weights are relative to a point
    that may lie 2^6 above or below the row's maximum, which in f16 makes half a subnormal step
    2^-25 * 2^6 of the largest weight."""
    outs, bounds = [], []
    u, H = plain.HALF_STEP[q.dtype], k.shape[1]
    group, D = q.shape[1] // H, q.shape[2]
    a = b = 0
    for lq, lkv in zip(q_lens, kv_lens):
        i, j = torch.arange(lq)[:, None], torch.arange(lkv)[None]
        see = j <= i
        if window:
            see &= (j > i - window) | (j < sinks)
        qq = q[a:a + lq].double()
        kk = k[b:b + lkv].double().repeat_interleave(group, 1)
        vv = v[b:b + lkv].double().repeat_interleave(group, 1)
        s = torch.matmul(qq.transpose(0, 1), kk.permute(1, 2, 0).contiguous()) * scale
        size = torch.matmul(qq.abs().transpose(0, 1), kk.abs().permute(1, 2, 0).contiguous()) * scale
        s = s.masked_fill(~see, float("-inf"))
        size = (size * see).amax(2, keepdim=True) if lkv else torch.zeros(q.shape[1], lq, 1, dtype=torch.float64)
        if lkv:
            p = torch.nan_to_num(torch.exp(s - s.amax(2, keepdim=True).clamp(min=-1e300)))
        else:
            p = torch.zeros(q.shape[1], lq, 0, dtype=torch.float64)
        l = p.sum(2, keepdim=True)
        inv = torch.where(l > 0, 1 / l, torch.zeros_like(l))
        vt = vv.transpose(0, 1)
        o = torch.matmul(p, vt) * inv
        spread = torch.matmul(p, vt.abs()) * inv
        n = see.sum(1).double().view(1, lq, 1)
        rel = 2 * u + 2 * size * (D + 4) * 2.0 ** -24 + 4 * 2.0 ** -22 + 2 * n * 2.0 ** -24
        bound = spread * rel + o.abs() * u
        total = torch.matmul(see.double().expand(q.shape[1], -1, -1), vt.abs()) * inv
        bound = bound + total * (2.0 ** -120 if q.dtype == torch.bfloat16 else 2.0 ** -19) + 2.0 ** -25 * (q.dtype == torch.float16)
        outs.append(o.transpose(0, 1)), bounds.append(bound.transpose(0, 1))
        a += lq
        b += lkv
    return torch.cat(outs), torch.cat(bounds)


def run_prefill(ops, q, k, v, q_lens, kv_lens, window, sinks, scale, out=None):
    cu_q = torch.tensor([0] + list(q_lens)).cumsum(0).to(torch.int32).cuda()
    cu_kv = torch.tensor([0] + list(kv_lens)).cumsum(0).to(torch.int32).cuda()
    got = ops.prefill_window(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_kv, max(q_lens), scale, window, sinks, out)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D", [(8, 2, 128), (4, 4, 64), (3, 1, 80), (2, 2, 256), (6, 2, 96), (4, 1, 32),
                                    (2, 1, 112), (2, 1, 120), (2, 1, 192)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 0), (64, 4), (100, 70), (300, 1), (5000, 3), (0, 0)])
def test_prefill_window(ops, dtype, Hq, H, D, window, sinks):
    g = torch.Generator().manual_seed(Hq * 1000 + D + window)
    lens = [1, 63, 64, 129, 2, 300]
    T = sum(lens)
    q, k, v = rows(g, T, Hq, D, dtype), rows(g, T, H, D, dtype), rows(g, T, H, D, dtype)
    got = run_prefill(ops, q, k, v, lens, lens, window, sinks, D ** -0.5)
    ref, bound = prefill_reference(q, k, v, lens, lens, window, sinks, D ** -0.5)
    plain.assert_within(got, ref, bound, f"window {window}, sinks {sinks}")


def test_prefill_window_longer_prompts(ops):
    """Windows that skip whole tiles, several workgroups per request, the XCD re-enumeration of eight
    (request, KV head) groups."""
    g = torch.Generator().manual_seed(5)
    Hq, H, D = 8, 4, 128
    lens = [1500, 777]
    T = sum(lens)
    q, k, v = (rows(g, T, h, D, torch.bfloat16) for h in (Hq, H, H))
    for window, sinks in ((256, 4), (128, 0), (257, 200), (64, 65), (700, 1400)):
        got = run_prefill(ops, q, k, v, lens, lens, window, sinks, D ** -0.5)
        ref, bound = prefill_reference(q, k, v, lens, lens, window, sinks, D ** -0.5)
        plain.assert_within(got, ref, bound, f"window {window}, sinks {sinks}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D", [(32, 8, 128), (40, 40, 96), (48, 8, 112)])
@pytest.mark.parametrize("window,sinks", [(64, 4), (250, 38), (251, 38), (400, 0), (0, 0)])
def test_prefill_window_launches_that_fill_the_chip(ops, dtype, Hq, H, D, window, sinks):
    """More than 256 workgroups: the shapes for rows that see few keys and for rows that see many, with 4, 1
    and 2 query heads side by side in a workgroup."""
    g = torch.Generator().manual_seed(Hq + D + window)
    lens = [513, 300, 290]
    T = sum(lens)
    q, k, v = rows(g, T, Hq, D, dtype), rows(g, T, H, D, dtype), rows(g, T, H, D, dtype)
    got = run_prefill(ops, q, k, v, lens, lens, window, sinks, D ** -0.5)
    pick = [0, Hq // H, Hq - 1]                        # the reference of every head would take minutes
    ref, bound = prefill_reference(q[:, pick], k[:, [p * H // Hq for p in pick]], v[:, [p * H // Hq for p in pick]],
                                   lens, lens, window, sinks, D ** -0.5)
    plain.assert_within(got[:, pick], ref, bound, f"window {window}, sinks {sinks}")
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("sinks", [0, 3])
def test_prefill_window_fewer_or_more_kv_rows(ops, sinks):
    """A pruned prompt (rows whose window lies past the last kv row see the sinks or nothing: zeros), more
    kv rows than queries, a request without kv rows, a request without queries."""
    g = torch.Generator().manual_seed(6)
    Hq, H, D = 4, 2, 64
    q_lens, kv_lens = [200, 50, 20, 0, 130], [70, 90, 0, 10, 130]
    q = rows(g, sum(q_lens), Hq, D, torch.float16)
    k, v = rows(g, sum(kv_lens), H, D, torch.float16), rows(g, sum(kv_lens), H, D, torch.float16)
    out = torch.full((sum(q_lens) + 9, Hq, D), 7.0, dtype=torch.float16, device="cuda")
    q = torch.cat([q, torch.full((9, Hq, D), float("nan"), dtype=torch.float16)])   # rows of no request
    got = run_prefill(ops, q, k, v, q_lens, kv_lens, 40, sinks, D ** -0.5, out)
    assert got is out and (out[-9:] == 7).all(), "rows behind the last request were touched"
    ref, bound = prefill_reference(q[:-9], k, v, q_lens, kv_lens, 40, sinks, D ** -0.5)
    plain.assert_within(got[:-9], ref, bound)
    if not sinks:
        assert (got[110:200] == 0).all() and (got[250:270] == 0).all()


def test_prefill_window_prefix_sums_past_the_rows(ops):
    """Prefix sums that reach past the rows of q or k are cut to them (never read or written past)."""
    g = torch.Generator().manual_seed(16)
    q, k, v = (rows(g, 90, h, 64, torch.bfloat16) for h in (4, 2, 2))
    cu = torch.tensor([0, 40, 90], dtype=torch.int32).cuda()
    far = torch.tensor([0, 40, 200], dtype=torch.int32).cuda()
    want = ops.prefill_window(q.cuda(), k.cuda(), v.cuda(), cu, cu, 50, 0.125, 20, 1)
    for a, b in ((far, far), (cu, far), (far, cu)):
        assert torch.equal(want, ops.prefill_window(q.cuda(), k.cuda(), v.cuda(), a, b, 160, 0.125, 20, 1))


def test_prefill_window_equals_causal_without_a_window(ops):
    g = torch.Generator().manual_seed(7)
    lens = [300, 41]
    q, k, v = (rows(g, 341, h, 128, torch.bfloat16).cuda() for h in (8, 2, 2))
    cu = torch.tensor([0, 300, 341], dtype=torch.int32).cuda()
    ref, bound = prefill_reference(q.cpu(), k.cpu(), v.cpu(), [300, 41], [300, 41], 0, 0, 128 ** -0.5)
    plain.assert_within(ops.prefill_causal(q, k, v, cu, cu, 300, 128 ** -0.5), ref, bound)
    a = ops.prefill_window(q, k, v, cu, cu, 300, 128 ** -0.5, 0, 0)
    for window, sinks in ((300, 0), (2 ** 31 - 1, 2 ** 31 - 1), (17, 300)):
        b = ops.prefill_window(q, k, v, cu, cu, 300, 128 ** -0.5, window, sinks)
        plain.assert_within(b, ref, bound, f"window {window}, sinks {sinks}")
    plain.assert_within(a, ref, bound)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_window_values_no_query_sees_through(ops, bad, D):
    """A NaN or an infinity in V (and in K) reaches the rows that see it, and only those: rows before it,
    rows whose window has left it, the next request."""
    g = torch.Generator().manual_seed(8)
    lens, window, sinks = [200, 70], 30, 2
    q, k, v = rows(g, 270, 4, D, torch.bfloat16), rows(g, 270, 2, D, torch.bfloat16), rows(g, 270, 2, D, torch.bfloat16)
    clean, bound = prefill_reference(q, k, v, lens, lens, window, sinks, D ** -0.5)
    at = 77
    v2 = v.clone()
    v2[at, 1, 5] = bad
    v2[199, 0] = bad            # the last row of the first request
    got = run_prefill(ops, q, k, v2, lens, lens, window, sinks, D ** -0.5).cpu().double()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:at + window, 2:, 5] = True
    hit[199, :2] = True
    assert not torch.isfinite(got[hit]).any()
    plain.assert_within(torch.where(hit, clean, got), clean, bound, "rows that do not see it")
    k2 = k.clone()
    k2[at, 0] = float("nan")
    got = run_prefill(ops, q, k2, v, lens, lens, window, sinks, D ** -0.5).cpu().double()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:at + window, :2] = True
    assert got[hit].isnan().all()
    plain.assert_within(torch.where(hit, clean, got), clean, bound, "rows that do not see it")


def test_prefill_window_strided_rows(ops):
    g = torch.Generator().manual_seed(9)
    Hq, H, D, T = 4, 2, 64, 150
    qkv = rows(g, T, Hq + 2 * H, D, torch.bfloat16).view(T, -1)
    cut = lambda t: (t[:, :Hq * D].unflatten(1, (Hq, D)), t[:, Hq * D:(Hq + H) * D].unflatten(1, (H, D)),  # noqa: E731
                     t[:, (Hq + H) * D:].unflatten(1, (H, D)))
    q, k, v = cut(qkv.cuda())
    wide = torch.full((T, Hq + 3, D), 3.0, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, T], dtype=torch.int32).cuda()
    ops.prefill_window(q, k, v, cu, cu, T, D ** -0.5, 17, 1, wide[:, :Hq])
    ref, bound = prefill_reference(*cut(qkv), [T], [T], 17, 1, D ** -0.5)
    plain.assert_within(wide[:, :Hq], ref, bound)
    assert (wide[:, Hq:] == 3).all()


def test_prefill_window_scores_that_creep_and_spike(ops):
    """The reference point of the weights moves late: scores that grow along the keys, and one spike."""
    g = torch.Generator().manual_seed(10)
    T, D = 400, 128
    q = torch.ones(T, 2, D).to(torch.float16)
    k = (torch.linspace(0, 30, T).view(T, 1, 1) * D ** -0.5 * torch.ones(1, 1, D)).to(torch.float16)
    k[211] = 4.0
    v = rows(g, T, 1, D, torch.float16)
    got = run_prefill(ops, q, k, v, [T], [T], 150, 4, D ** -0.5)
    ref, bound = prefill_reference(q, k, v, [T], [T], 150, 4, D ** -0.5)
    plain.assert_within(got, ref, bound)


# ------------------------------------------------------------------ decode over 16-bit pages
def pool(g, lens, H, D, bs, dtype, spare=4):
    counts = [-(-n // bs) for n in lens]
    nb = sum(counts) + spare
    kc = torch.randn(nb, H, D // 8, bs, 8, generator=g).to(dtype)
    vc = torch.randn(nb, H, D, bs, generator=g).to(dtype)
    ids = torch.randperm(nb, generator=g)[:sum(counts)].to(torch.int32)
    t = torch.full((len(lens), max(1, max(counts))), -3, dtype=torch.int32)
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        t[i, :c] = ids[at:at + c]
        at += c
        if n % bs:      # slots behind the sequence hold anything
            kc[t[i, c - 1].long(), :, :, n % bs:] = float("nan")
            vc[t[i, c - 1].long(), :, :, n % bs:] = float("inf")
    return kc, vc, t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D,bs", [(32, 8, 128, 16), (12, 12, 64, 16), (8, 2, 128, 8), (8, 1, 128, 32),
                                       (5, 1, 80, 16), (4, 2, 96, 8), (2, 1, 112, 32), (2, 1, 120, 16),
                                       (40, 2, 64, 16), (16, 1, 192, 8), (6, 2, 256, 16), (4, 2, 32, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 5), (100, 64), (1000, 4)])
def test_decode_window(ops, dtype, Hq, H, D, bs, window, sinks):
    g = torch.Generator().manual_seed(Hq + D + bs + window)
    lens = [1, bs, 0, 31, 32, 33, 200, 517]
    kc, vc, t = pool(g, lens, H, D, bs, dtype)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, len(lens), Hq, D, dtype)
    kz, vz = torch.nan_to_num(kc), torch.nan_to_num(vc, posinf=0.0)
    ref, bound = plain.decode(q, kz, vz, None, t, ln, window, sinks, D ** -0.5)
    for s, n in enumerate(lens):
        seen = plain.visible(n, window, sinks)
        for j in range(-(-n // bs)):
            if not seen[j * bs:(j + 1) * bs].any():
                t[s, j] = 1 << 30
    out = torch.full_like(q, float("nan")).cuda()
    ops.paged_attention_window(out, q.cuda(), kc.cuda(), vc.cuda(), H, D ** -0.5, t.cuda(), ln.cuda(), bs,
                               max(lens), window, sinks)
    plain.assert_within(out, ref, bound, f"window {window}, sinks {sinks}")
    assert (out[2] == 0).all()
    ops.check_device_diagnostics()


def test_decode_window_negative_scale_and_hidden_nan(ops):
    """Scores of either sign of scale; NaN keys and values left of the window inside a visible block."""
    g = torch.Generator().manual_seed(21)
    kc, vc, t = pool(g, [90], 2, 64, 16, torch.bfloat16)
    q, ln = rows(g, 1, 4, 64, torch.bfloat16), torch.tensor([90], dtype=torch.int32)
    for scale in (-0.3, 0.0, 0.125):
        ref, bound = plain.decode(q, torch.nan_to_num(kc), torch.nan_to_num(vc, posinf=0.0), None, t, ln, 35, 3, scale)
        k2, v2 = kc.clone(), vc.clone()
        for blk, slots in ((int(t[0, 0]), slice(3, None)), (int(t[0, 3]), slice(0, 7))):
            k2[blk, :, :, slots] = float("nan")
            v2[blk, :, :, slots] = float("nan")
        out = torch.empty_like(q).cuda()
        ops.paged_attention_window(out, q.cuda(), k2.cuda(), v2.cuda(), 2, scale, t.cuda(), ln.cuda(), 16, 90, 35, 3)
        plain.assert_within(out, ref, bound, f"scale {scale}")


@pytest.mark.parametrize("S,Hq,H,D,longest", [
    (9, 8, 8, 128, 1500),     # one workgroup of many waves per sequence and head, several tiles per wave
    (34, 4, 4, 64, 5000),     # three splits
    (17, 12, 12, 64, 5000),   # two splits of small tiles
    (50, 12, 6, 32, 2500),    # two splits of more than 256 workgroups
    (25, 8, 8, 96, 9000),     # none
    (5, 8, 8, 80, 8000)])     # a workgroup per compute unit
@pytest.mark.parametrize("window,sinks", [(0, 0), (1200, 3)])
def test_decode_window_launch_shapes(ops, S, Hq, H, D, longest, window, sinks):
    """The launch is shaped by the longest sequence that may come; the ones that do are ragged, most of
    them with nothing for most of the waves and splits."""
    g = torch.Generator().manual_seed(S + D)
    lens = [int(torch.randint(0, 60, (), generator=g)) for _ in range(S)]
    lens[1], lens[S - 1], lens[2] = 1490, 777, 0
    kc, vc, t = pool(g, lens, H, D, 16, torch.bfloat16)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, S, Hq, D, torch.bfloat16)
    ref, bound = plain.decode(q, torch.nan_to_num(kc), torch.nan_to_num(vc, posinf=0.0), None, t, ln, window, sinks,
                              D ** -0.5)
    out = torch.full_like(q, float("nan")).cuda()
    ops.paged_attention_window(out, q.cuda(), kc.cuda(), vc.cuda(), H, D ** -0.5, t.cuda(), ln.cuda(), 16, longest,
                               window, sinks)
    plain.assert_within(out, ref, bound, f"{S} x {H}, up to {longest}")
    assert (out[2] == 0).all()
    ops.check_device_diagnostics()
