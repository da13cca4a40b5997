"""The 8-bit paged cache on the GPU where its rules meet their ends: blocks of scale 0 and of scales that are
no powers of two, f16 weights beside value blocks of zeros, scores far from zero, waves that take many tiles."""
import pytest
import torch

import plain_window as plain
from test_gpu_8bit_cache import FORMATS, filled, garbage_cache, rows, run_attention, same_bits, tables_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import vllm_paged_compression_amd as pkg
    import vllm_paged_compression_amd.ops as ops
    pkg.load_library()
    return ops


def append(key, value, kc, vc, sc, t, lens, fmt):
    """One row per sequence, from the definition, in place on CPU tensors: the block takes s = max(s_old, need), its
    older codes become rn(code * s_old / s), also from s_old = 0; quotients are rounded to f32 first."""
    bs = vc.shape[3]
    for s, n in enumerate(lens.tolist()):
        b, o = int(t[s, (n - 1) // bs]), (n - 1) % bs
        for which, (new, cache, get) in enumerate(((key, kc, plain.k_rows), (value, vc, plain.v_rows))):
            codes, block = get(cache, b), cache[b].clone()
            for h in range(new.shape[1]):
                x = new[s, h].double()
                finite = x[torch.isfinite(x)].abs()
                old = float(sc[b, h, which]) if o else 0.0
                scale = max(old, plain.need_scale(float(finite.max()) if finite.numel() else 0.0, fmt))
                if o and scale > old:
                    plain.put(block, h, 0, plain.encode(codes[h, :o] * (old / scale), fmt), which)
                quotient = (x / scale).float().double() if scale else x
                plain.put(block, h, o, plain.encode(quotient, fmt)[None], which)
                sc[b, h, which] = scale
            cache[b] = block


def same_values(a, b):
    a, b = a.cpu().float(), b.float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ------------------------------------------------------------------ blocks whose scale is 0
@pytest.mark.parametrize("how", ["write", "chunk", "step"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D,bs,older", [(4, 2, 64, 16, 1), (8, 1, 128, 8, 7), (2, 2, 80, 32, 19), (4, 2, 256, 16, 3),
                                             (20, 1, 64, 16, 2)])
def test_joining_a_block_of_zeros_and_infinities(ops, how, fmt, dtype, Hq, H, D, bs, older):
    """Rows of zeros, infinities (the largest code) and NaN leave a block with scale 0: every element that is no NaN
    reads as 0.  It still does after a finite row has given the block a scale."""
    g = torch.Generator().manual_seed(older + D)
    kc, vc, sc = garbage_cache(g, 9, H, D, bs, fmt)
    lens = [older, bs + older]                       # the block is the sequence's first one, and its second
    t = tables_for(g, 9, [3 * bs, 3 * bs], bs)
    T = sum(lens)
    k, v = rows(g, T, H, D, dtype), rows(g, T, H, D, dtype)
    for x in (k, v):
        for first in (0, T - older):
            x[first:first + older] = 0
            x[first, 0, 3], x[first + older - 1, H - 1, 7] = float("inf"), float("-inf")
    v[0, 0, 5] = float("nan")
    cu, ln = torch.tensor([0, lens[0], T], dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    dev = [x.cuda() for x in (kc, vc, sc)]
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)    # (these writes begin their blocks)
    ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), ln.cuda(), cu.cuda(), max(lens), fmt)
    assert float(dev[2][t[0, 0].long()].max()) == 0 and float(dev[2][t[1, 1].long()].max()) == 0
    assert all(same_values(a, b) for a, b in zip(dev, (kc, vc, sc)))

    for step in range(2):                            # the second one joins a block that has a scale
        ln = ln + 1
        k, v = (torch.ones(2, H, D, dtype=dtype) if step == 0 else rows(g, 2, H, D, dtype, 9.0) for _ in range(2))
        k[1, 0, ::2], v[1, 0, ::2] = 0, 0
        args = (k.cuda(), v.cuda(), *dev)
        if how == "step":
            q = rows(g, 2, Hq, D, dtype)
            out = torch.empty_like(q).cuda()
            ops.decode_step_8bit(out, q.cuda(), *args, H, D ** -0.5, t.cuda(), ln.cuda(), bs, 3 * bs, fmt)
        else:
            cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda() if how == "chunk" else None
            ops.reshape_and_cache_8bit(*args, t.cuda(), ln.cuda(), cu, 1, fmt)
        append(k, v, kc, vc, sc, t, ln, fmt)
        assert same_bits(dev[2], sc), f"step {step}: scales"
        for name, a, b in zip(("key codes", "value codes"), dev, (kc, vc)):
            assert same_values(a, b), f"step {step}: {name}"
        if how == "step":
            # (the NaN of sequence 0 reaches its outputs)
            ref, bound = plain.decode(q[1:], kc, vc, sc, t[1:], ln[1:], 0, 0, D ** -0.5)
            plain.assert_within(out[1:], ref, bound, f"step {step}")
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
def test_joining_a_block_that_a_caller_gave_scale_zero(ops, fmt):
    """Any codes under a scale of 0 (a cache made elsewhere) are zeros, whatever joins them."""
    g = torch.Generator().manual_seed(5)
    H, D, bs, S = 2, 64, 16, 3
    kc, vc, sc, t = filled(g, [9, 3, 15], H, D, bs, fmt)
    sc[t[:, 0].long()] = 0.0
    ln = torch.tensor([10, 4, 16], dtype=torch.int32)
    k, v, q = rows(g, S, H, D, torch.bfloat16), rows(g, S, H, D, torch.bfloat16), rows(g, S, 4, D, torch.bfloat16)
    k[2], v[2] = 0, 0                               # nothing to scale: the codes stay as they are
    out, dev = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0, step=(k, v))
    append(k, v, kc, vc, sc, t, ln, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, t, ln, 0, 0, D ** -0.5))


# ------------------------------------------------------------------ blocks whose scale is no power of two
@pytest.mark.parametrize("how", ["write", "step"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_joining_blocks_of_any_scale(ops, how, fmt, dtype):
    """Scales of a cache made elsewhere: x / s is rounded once to f32 (x times a rounded 1 / s falls off the ties of
    these rows), also where 1 / s is past f32's largest number."""
    g = torch.Generator().manual_seed(6)
    H, D, bs, S = 2, 64, 16, 60
    # x / s lies on the tie `half` in f32, x * (1 / s) next to it
    x = torch.arange(128.0, 256.0)[:, None]
    half = torch.arange(8) + 0.5 if fmt == "int8" else torch.arange(17.0, 32.0, 2)[:8]
    scale = x / half
    apart = (x / scale == half) & (x * (1 / scale) != half)
    at = apart.nonzero()
    at = at[torch.randperm(len(at), generator=g)[:S - 3]]
    assert len(at) == S - 3
    kc, vc, sc, t = filled(g, [5] * S, H, D, bs, fmt)
    k, v = torch.zeros(S, H, D, dtype=dtype), torch.zeros(S, H, D, dtype=dtype)
    for s, (i, j) in enumerate(at.tolist()):
        sc[t[s, 0].long()] = scale[i, j]
        k[s], v[s, :, 3:] = float(x[i]), -float(x[i])
    for s, tiny in zip(range(S - 3, S), (1e-39, 2.0 ** -149, 2.0 ** -130)):
        sc[t[s, 0].long()] = tiny                        # rows of zeros leave it
    sc[t[0, 0].long(), :, 0], k[0] = 0.0, 0              # nothing to divide beside a quotient
    ln = torch.full((S,), 6, dtype=torch.int32)
    if how == "step":
        q = rows(g, S, 4, D, dtype)
        _, dev = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0, step=(k, v))
    else:
        dev = [x.cuda() for x in (kc, vc, sc)]
        ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), ln.cuda(), None, 1, fmt)
    append(k, v, kc, vc, sc, t, ln, fmt)
    for name, a, b in zip(("key codes", "value codes", "scales"), dev, (kc, vc, sc)):
        assert same_bits(a, b), name


# ------------------------------------------------------------------ f16 weights
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gap", [5.0, 60.0, 80.0, 88.0, 90.0, 200.0, 3000.0])
@pytest.mark.parametrize("where", ["same tile", "earlier tile", "later tile"])
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_f16_peak_on_value_rows_of_zeros(ops, fmt, gap, where, bs):
    """The heaviest keys lie in a block whose values are zeros (scale 0), `gap` nats above the rest.  A launch shaped
    for one tile walks these nine tiles of 64 tokens with four waves: wave 0 takes tiles 0, 4 and 8."""
    g = torch.Generator().manual_seed(bs)
    H, D, n = 1, 64, 9 * 64
    at = {"same tile": 4 * 64 + 32, "earlier tile": 0, "later tile": 8 * 64}[where]
    kc, vc, sc = garbage_cache(g, n // bs + 2, H, D, bs, fmt)
    t = tables_for(g, n // bs + 2, [n], bs)
    k, v = 0.02 * rows(g, n, H, D, torch.float16), rows(g, n, H, D, torch.float16)
    v[at:at + 32] = 0
    q = torch.ones(1, 4, D, dtype=torch.float16)
    k[at + 3] = gap * D ** 0.5 / D                    # q . k * scale = gap
    cu, ln = torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, 0, 0, D ** -0.5)
    for max_len in (64, n):
        out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0, max_len=max_len)
        plain.assert_within(out, ref, bound, f"launch shaped for {max_len} tokens")
    new = torch.zeros(1, H, D, dtype=torch.float16)
    # the step that starts a block with a row of zeros and a peak
    wide = torch.cat([t, torch.tensor([[b for b in range(n // bs + 2) if b not in t[0].tolist()][:1]], dtype=torch.int32)], 1)
    peak = new + k[at + 3]
    out, dev = run_attention(ops, q, kc, vc, sc, wide, ln + 1, fmt, 0, 0, step=(peak, new), max_len=64)
    append(peak, new, kc, vc, sc, wide, ln + 1, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, wide, ln + 1, 0, 0, D ** -0.5), "step")


# ------------------------------------------------------------------ many tiles per wave, launch shapes
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("order", ["falling", "rising", "both"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_tiles_per_wave(ops, fmt, order, dtype):
    """45 tiles on four waves, scores and value scales that rise or fall by turns along the sequence: both reference
    points of f16 weights move often, and in unlike directions."""
    g = torch.Generator().manual_seed(14)
    H, D, bs, n = 2, 64, 16, 45 * 64 - 11
    kc, vc, sc = garbage_cache(g, n // bs + 4, H, D, bs, fmt)
    t = tables_for(g, n // bs + 4, [n], bs)
    k, v = rows(g, n, H, D, dtype, 0.3), rows(g, n, H, D, dtype)
    x = torch.linspace(0, 1, n)
    ramp = {"falling": 1 - x, "rising": x, "both": (2 * x - 1).abs()}[order]
    k = (k.float() + (25 * ramp * D ** -0.5).view(n, 1, 1)).to(dtype)             # scores move by 25 nats
    v = (v.float() * torch.exp2(8 * (0.5 - ramp) + 3 * torch.sin(40 * x)).view(n, 1, 1)).to(dtype)
    q = torch.ones(1, 8, D, dtype=dtype) + 0.2 * rows(g, 1, 8, D, dtype)
    cu, ln = torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    for window, sinks in ((0, 0), (2000, 100)):
        ref, bound = plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5)
        for max_len in (64, n, 1 << 20):
            out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, max_len=max_len)
            plain.assert_within(out, ref, bound, f"window {window}, launch shaped for {max_len} tokens")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("S,Hq,H,D,longest", [(9, 8, 8, 128, 3000), (34, 4, 4, 64, 8000), (17, 12, 12, 64, 8000),
                                              (50, 6, 6, 32, 2500), (25, 8, 8, 96, 9000), (5, 8, 8, 80, 9000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1200, 3)])
def test_f16_launch_shapes(ops, fmt, S, Hq, H, D, longest, window, sinks):
    """The launch shapes with f16 rows: partials whose weights have their own reference points, joined."""
    g = torch.Generator().manual_seed(S + D)
    lens = [int(torch.randint(1, 60, (), generator=g)) for _ in range(S)]
    lens[1], lens[S - 1], lens[2] = 1490, 777, 0
    bs, dtype = 16, torch.float16
    kc, vc, sc, t = filled(g, [n + 1 if n else 0 for n in lens], H, D, bs, fmt, dtype)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, S, Hq, D, dtype)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, max_len=longest)
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5), "attention")
    k, v = rows(g, S, H, D, dtype, 3.0), rows(g, S, H, D, dtype, 3.0)
    ln = torch.where(ln > 0, ln + 1, ln)
    out, dev = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, step=(k, v), max_len=longest)
    plain.write(k, v, kc, vc, sc, t, ln, None, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5), "step")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1024 * 64 - 5, 1024 * 64 + 70])
def test_one_long_request_on_one_kv_head(ops, dtype, n):
    """Both sides of 1024 tiles of one (sequence, KV head), where the launch changes its shape."""
    g = torch.Generator().manual_seed(15)
    D, bs = 32, 32
    kc, vc, sc, t = filled(g, [n], 1, D, bs, "int8", dtype)
    ln = torch.tensor([n], dtype=torch.int32)
    q = rows(g, 1, 4, D, dtype)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, "int8", 0, 0)
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, t, ln, 0, 0, D ** -0.5))


# ------------------------------------------------------------------ scores far from zero
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e9, 1e10, 1e25, 1e33])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_scores_far_from_zero(ops, fmt, dtype, size, sign):
    """All scores near `sign * size`, one key ahead of the others by more than f32's step there: the output is the
    value of that key, however far the scores are from zero."""
    g = torch.Generator().manual_seed(16)
    H, D, bs, n, ahead = 1, 64, 16, 200, 77
    kc, vc, sc = garbage_cache(g, 16, H, D, bs, fmt)
    t = tables_for(g, 16, [n], bs)
    k, v = torch.full((n, H, D), 1.0, dtype=dtype), rows(g, n, H, D, dtype)
    k[ahead] = 1.5 if sign > 0 else 0.5
    cu, ln = torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    sc[t[0].long(), :, 0] *= size / 8                  # K's scales carry the size
    q = torch.full((1, 2, D), sign, dtype=dtype)
    block, slot = int(t[0, ahead // bs]), ahead % bs
    want = (plain.v_rows(vc, block)[0, slot] * float(sc[block, 0, 1])).to(dtype)
    for max_len in (64, n, 1 << 16):
        out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0, max_len=max_len)
        assert torch.equal(out.cpu(), want.expand(1, 2, D)), f"launch shaped for {max_len} tokens"
