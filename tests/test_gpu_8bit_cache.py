"""The 8-bit paged cache on the GPU: writes (codes and scales bit for bit), decode attention and the
decode step against a plain implementation in 64 bits."""
import pytest
import torch

import plain_window as plain

pytestmark = pytest.mark.gpu

FORMATS = ["fp8", "int8"]


@pytest.fixture(scope="module")
def ops():
    import vllm_paged_compression_amd as pkg
    import vllm_paged_compression_amd.ops as ops
    pkg.load_library()
    return ops


def rows(g, n, heads, D, dtype, size=1.0):
    return (torch.randn(n, heads, D, generator=g) * torch.exp(0.7 * torch.randn(heads, D, generator=g)) * size).to(dtype)


def garbage_cache(g, nb, H, D, bs, fmt):
    """A pool as recycled memory leaves it: any byte (NaN codes included), any scale."""
    kc = torch.randint(0, 256, (nb, H, D // 16, bs, 16), generator=g, dtype=torch.uint8)
    vc = torch.randint(0, 256, (nb, H, D, bs), generator=g, dtype=torch.uint8)
    sc = torch.rand(nb, H, 2, generator=g) * 1e30
    sc[::3] = float("nan")
    sc[1::3, :, 1] = float("inf")
    return kc.view(plain.CODE_DTYPE[fmt]), vc.view(plain.CODE_DTYPE[fmt]), sc


def tables_for(g, nb, lens, bs, width=None):
    counts = [-(-n // bs) for n in lens]
    ids = torch.randperm(nb, generator=g)[:sum(counts)].to(torch.int32)
    t = torch.full((len(lens), width or max(1, max(counts))), -7, dtype=torch.int32)   # unused entries: no block
    at = 0
    for i, c in enumerate(counts):
        t[i, :c] = ids[at:at + c]
        at += c
    return t


def filled(g, lens, H, D, bs, fmt, dtype=torch.bfloat16, spare=5):
    """A pool with the sequences written by the plain implementation; every other slot is garbage."""
    nb = sum(-(-n // bs) for n in lens) + spare
    kc, vc, sc = garbage_cache(g, nb, H, D, bs, fmt)
    t = tables_for(g, nb, lens, bs)
    cu = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)
    T = int(cu[-1])
    plain.write(rows(g, T, H, D, dtype), rows(g, T, H, D, dtype), kc, vc, sc, t,
                torch.tensor(lens, dtype=torch.int32), cu, fmt)
    return kc, vc, sc, t


def same_bits(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ------------------------------------------------------------------ writes
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,bs", [(8, 128, 16), (3, 64, 8), (1, 80, 16), (2, 96, 32), (2, 112, 8),
                                    (1, 192, 16), (2, 256, 32), (5, 32, 16)])
def test_write_prompts_then_steps(ops, fmt, dtype, H, D, bs):
    """Ragged prompts into recycled blocks, a second chunk that joins half-filled blocks, then single
    rows, some far larger than what their block holds: codes and scales bit for bit."""
    g = torch.Generator().manual_seed(H * 1000 + D + bs)
    lens = [1, bs - 1, bs, 3 * bs + 5, 2]
    grow = [0, bs + 3, 1, 7, 2 * bs]
    total = [a + b + 4 for a, b in zip(lens, grow)]
    nb = sum(-(-n // bs) for n in total) + 3
    kc, vc, sc = garbage_cache(g, nb, H, D, bs, fmt)
    t = tables_for(g, nb, total, bs)
    dev = [x.cuda() for x in (kc, vc, sc)]
    now = [0] * len(lens)
    for step, add in enumerate([lens, grow] + [[1] * len(lens)] * 4):
        now = [a + b for a, b in zip(now, add)]
        cu = torch.tensor([0] + add).cumsum(0).to(torch.int32)
        T = int(cu[-1])
        size = 2.0 ** (3 * step)
        k, v = rows(g, T, H, D, dtype, size), rows(g, T, H, D, dtype, 1 / size)
        ln = torch.tensor(now, dtype=torch.int32)
        one = max(add) == 1 and min(add) == 1
        plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
        ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), ln.cuda(), None if one else cu.cuda(),
                                   max(add), fmt)
        torch.cuda.synchronize()
        for name, got, want in zip(("key codes", "value codes", "scales"), dev, (kc, vc, sc)):
            assert same_bits(got, want), f"step {step}: {name}"
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_special_values(ops, fmt):
    """Zeros, subnormals, the ends of the range, values next to a power of two times FMAX, infinities
    and NaN, every one in a block of its own."""
    bs, H, D = 16, 1, 32
    top = plain.FMAX[fmt]
    fills = [0.0, -0.0, 1e-40, 9.2e-41, 1e-30, top, top * 1.0078125, top / 2, 2 * top, 3.3e38, -1.0]
    T = len(fills) * bs
    k = torch.zeros(T, H, D, dtype=torch.bfloat16)
    for i, f in enumerate(fills):
        k[i * bs:(i + 1) * bs] = torch.linspace(-1, 1, bs * D).view(bs, 1, D).to(torch.bfloat16) * torch.tensor(f, dtype=torch.bfloat16)
        k[i * bs, 0, 3] = f
    v = k.clone()
    v[5 * bs, 0, 0], v[6 * bs, 0, 1], v[7 * bs, 0, 2] = float("inf"), float("-inf"), float("nan")
    v[:bs] = float("inf")       # a block without a finite value
    nb = len(fills) + 1
    g = torch.Generator().manual_seed(1)
    kc, vc, sc = garbage_cache(g, nb, H, D, bs, fmt)
    t = torch.arange(len(fills), dtype=torch.int32)[None]
    ln, cu = torch.tensor([T], dtype=torch.int32), torch.tensor([0, T], dtype=torch.int32)
    dev = [x.cuda() for x in (kc, vc, sc)]
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), ln.cuda(), cu.cuda(), T, fmt)
    assert torch.equal(dev[2].cpu()[:-1], sc[:-1])
    for got, want in zip(dev[:2], (kc, vc)):
        got, want = got.cpu()[:-1].float(), want[:-1].float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_write_uint8_storage_strided_rows_and_no_rows(ops):
    """fp8 codes in uint8 tensors, rows cut out of a fused activation, sequences without rows."""
    g = torch.Generator().manual_seed(2)
    H, D, bs = 2, 64, 16
    lens = torch.tensor([20, 0, 33], dtype=torch.int32)
    cu = torch.tensor([0, 20, 20, 20 + 5], dtype=torch.int32)
    kc, vc, sc = garbage_cache(g, 8, H, D, bs, "fp8")
    t = tables_for(g, 8, [20, 0, 33], bs)
    sc[t[2, :3].long()] = 2.0 ** -3
    qkv = rows(g, 25, 3 * H, D, torch.bfloat16).view(25, -1).cuda()
    k, v = qkv[:, H * D:2 * H * D].unflatten(1, (H, D)), qkv[:, 2 * H * D:].unflatten(1, (H, D))
    dev = [x.view(torch.uint8).cuda() for x in (kc, vc)] + [sc.cuda()]
    plain.write(k.cpu(), v.cpu(), kc, vc, sc, t, lens, cu, "fp8")
    ops.reshape_and_cache_8bit(k, v, *dev, t.cuda(), lens.cuda(), cu.cuda(), 3, "fp8_e4m3")   # max_q_len too small: only sizes the grid
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    before = [x.clone() for x in dev]
    ops.reshape_and_cache_8bit(k[:0], v[:0], *dev, t.cuda(), lens.cuda(), torch.zeros(4, dtype=torch.int32).cuda(), 0, "fp8")
    assert all(same_bits(a, b.cpu()) for a, b in zip(dev, before))


def test_write_skips_what_does_not_fit_and_reports_it(ops):
    """More rows than the length, rows past the tensor, a length past the table, a block outside the
    pool: those sequences (that block) are left alone, the others are written."""
    g = torch.Generator().manual_seed(3)
    H, D, bs, fmt = 2, 32, 16, "int8"
    ops.device_diagnostics()
    lens = torch.tensor([5, 2, 40, 20], dtype=torch.int32)
    cu = torch.tensor([0, 5, 8, 12, 32], dtype=torch.int32)
    t = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 99]], dtype=torch.int32)
    kc, vc, sc = garbage_cache(g, 8, H, D, bs, fmt)
    dev = [x.cuda() for x in (kc, vc, sc)]
    k, v = rows(g, 32, H, D, torch.float16), rows(g, 32, H, D, torch.float16)
    plain.write(k, v, kc, vc, sc, t, lens, cu, fmt)
    ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), lens.cuda(), cu.cuda(), 20, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    assert ops.device_diagnostics() == ops.DIAG_BLOCK_ID | ops.DIAG_APPEND_MISMATCH


# ------------------------------------------------------------------ attention
def run_attention(ops, q, kc, vc, sc, t, lens, fmt, window, sinks, max_len=None, step=None):
    dev = [x.cuda() for x in (kc, vc, sc)]
    out = torch.full_like(q, float("nan")).cuda()
    D, bs, H = vc.shape[2], vc.shape[3], vc.shape[1]
    args = (H, D ** -0.5, t.cuda(), lens.cuda(), bs, max_len or max(1, int(lens.max())), fmt, window, sinks)
    if step is None:
        ops.paged_attention_8bit(out, q.cuda(), *dev, *args)
    else:
        ops.decode_step_8bit(out, q.cuda(), step[0].cuda(), step[1].cuda(), *dev, *args)
    torch.cuda.synchronize()
    return out, dev


GEOMETRY = [(32, 8, 128, 16), (12, 12, 64, 16), (8, 1, 128, 8), (8, 2, 128, 32), (5, 1, 80, 16), (4, 2, 96, 8),
            (4, 4, 112, 32), (40, 2, 64, 16), (16, 1, 192, 16), (6, 2, 256, 8), (2, 1, 256, 32), (4, 2, 32, 8),
            (4, 2, 32, 32)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D,bs", GEOMETRY)
def test_attention_over_the_whole_cache(ops, fmt, dtype, Hq, H, D, bs):
    g = torch.Generator().manual_seed(Hq + D + bs)
    lens = [1, bs, 0, 63, 64, 65, 200, 129]
    kc, vc, sc, t = filled(g, lens, H, D, bs, fmt)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, len(lens), Hq, D, dtype)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, 0, 0, D ** -0.5)
    plain.assert_within(out, ref, bound, "whole cache")
    assert (out[2] == 0).all()
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (50, 0), (64, 64), (100, 37), (1000, 4), (130, 1000)])
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_attention_through_a_window(ops, fmt, window, sinks, bs):
    """Window and sinks ending inside blocks and tiles, overlapping, longer than the sequence; blocks
    that hold no visible token have been given away (their table entries name no block)."""
    g = torch.Generator().manual_seed(window * 100 + sinks + bs)
    Hq, H, D = 8, 2, 64
    lens = [1, 15, 64, 129, 300, 517]
    kc, vc, sc, t = filled(g, lens, H, D, bs, fmt)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, len(lens), Hq, D, torch.bfloat16)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5)
    for s, n in enumerate(lens):
        seen = plain.visible(n, window, sinks)
        for j in range(-(-n // bs)):
            if not seen[j * bs:(j + 1) * bs].any():
                t[s, j] = -1
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks)
    plain.assert_within(out, ref, bound, f"window {window}, sinks {sinks}")
    ops.check_device_diagnostics()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_blocks_of_very_unlike_scales(ops, fmt, dtype):
    """Value blocks 2^12 apart, blocks of zeros, and the attention on the small ones: the weights of
    f16 keep their bits whatever the scale in front of V is."""
    g = torch.Generator().manual_seed(9)
    H, D, bs, n = 2, 64, 16, 160
    kc, vc, sc = garbage_cache(g, 12, H, D, bs, fmt)
    t = tables_for(g, 12, [n], bs)
    k, v = rows(g, n, H, D, dtype), rows(g, n, H, D, dtype)
    for j in range(n // bs):
        v[j * bs:(j + 1) * bs] = (v[j * bs:(j + 1) * bs].float() * 2.0 ** (6 if j % 3 == 0 else -6)).to(dtype)
    v[5 * bs:6 * bs] = 0
    k[3 * bs:4 * bs] = 0
    q = rows(g, 1, 4, D, dtype)
    k[4 * bs + 3] = q[0, 0] * 0.5                                          # a peak on a small block
    cu, ln = torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, 0, 0)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, 0, 0, D ** -0.5)
    plain.assert_within(out, ref, bound, "unlike scales")


def test_attention_arbitrary_scales(ops):
    """Scales that are no powers of two (a cache made elsewhere)."""
    g = torch.Generator().manual_seed(10)
    kc, vc, sc, t = filled(g, [100], 2, 128, 16, "int8")
    sc = torch.where(torch.isfinite(sc) & (sc < 1e20), sc * (0.5 + torch.rand(sc.shape, generator=g)), sc)
    q, ln = rows(g, 1, 8, 128, torch.float16), torch.tensor([100], dtype=torch.int32)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, "int8", 0, 0)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, 0, 0, 128 ** -0.5)
    plain.assert_within(out, ref, bound, "arbitrary scales")


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_attention_long_sequences_few_and_many(ops, window, sinks):
    """The split over the keys (few rows) and whole rows per workgroup (many) agree with the formula."""
    g = torch.Generator().manual_seed(11)
    H, D, bs = 1, 128, 16
    kc, vc, sc, t = filled(g, [5003], H, D, bs, "fp8")
    for seqs in (1, 3, 20, 300):
        ln = torch.full((seqs,), 5003, dtype=torch.int32)
        q = rows(g, 3, 4, D, torch.bfloat16)[torch.arange(seqs) % 3].contiguous()
        out, _ = run_attention(ops, q, kc, vc, sc, t.expand(seqs, -1).contiguous(), ln, "fp8", window, sinks)
        n = min(seqs, 3)
        ref, bound = plain.decode(q[:n], kc, vc, sc, t.expand(n, -1), ln[:n], window, sinks, D ** -0.5)
        plain.assert_within(out[:n], ref, bound, f"{seqs} sequences")
        if seqs > 3:
            assert torch.equal(out[3:], out[:3][torch.arange(3, seqs) % 3]), "a row's result hangs on its place"


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_and_step_many_short_sequences(ops, fmt):
    """Launches of 100 workgroups with some tiles each (the wide workgroups), attention and step."""
    g = torch.Generator().manual_seed(13)
    H, D, bs, S = 1, 64, 16, 100
    lens = [850 + 5 * i % 61 for i in range(S)]
    kc, vc, sc, t = filled(g, [912] * 3, H, D, bs, fmt, spare=S + 5)
    full = t[torch.arange(S) % 3].clone()
    # the sequences share their full blocks; each has a last block of its own
    free = torch.tensor([b for b in range(vc.shape[0]) if b not in set(t.flatten().tolist())], dtype=torch.int32)
    for s, n in enumerate(lens):
        own, old = int(free[s]), int(full[s, n // bs])
        kc[own], vc[own], sc[own] = kc[old], vc[old], sc[old]
        full[s, n // bs] = own
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, S, 4, D, torch.bfloat16)
    out, _ = run_attention(ops, q, kc, vc, sc, full, ln, fmt, 0, 0)
    ref, bound = plain.decode(q[:8], kc, vc, sc, full, ln[:8], 0, 0, D ** -0.5)
    plain.assert_within(out[:8], ref, bound, "attention")
    k, v = rows(g, S, H, D, torch.bfloat16, 3.0), rows(g, S, H, D, torch.bfloat16, 3.0)
    ln = ln + 1
    out, dev = run_attention(ops, q, kc, vc, sc, full, ln, fmt, 0, 0, step=(k, v))
    plain.write(k, v, kc, vc, sc, full, ln, None, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    ref, bound = plain.decode(q[:8], kc, vc, sc, full, ln[:8], 0, 0, D ** -0.5)
    plain.assert_within(out[:8], ref, bound, "step")


def test_attention_reports_bad_blocks_and_lengths(ops):
    """A visible table entry outside the pool counts as not visible, a length past the table row is cut
    to it; both are reported."""
    g = torch.Generator().manual_seed(12)
    H, D, bs = 2, 64, 16
    kc, vc, sc, t = filled(g, [100, 48], H, D, bs, "fp8")
    q = rows(g, 2, 4, D, torch.bfloat16)
    ln = torch.tensor([100, 48], dtype=torch.int32)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, 32, 16, D ** -0.5)   # blocks 0 and from 68 on
    bad = t.clone()
    bad[0, 1:4] = torch.tensor([10 ** 6, -5, 99])
    ops.device_diagnostics()
    out, _ = run_attention(ops, q, kc, vc, sc, bad, ln, "fp8", 32, 16)
    plain.assert_within(out, ref, bound, "stale entries outside the window")
    assert ops.device_diagnostics() == 0
    bad = t.clone()
    bad[0, 2] = 10 ** 6
    out, _ = run_attention(ops, q, kc, vc, sc, bad, ln, "fp8", 0, 0)
    assert ops.device_diagnostics() == ops.DIAG_BLOCK_ID
    k, v, vs = plain.gather(kc, vc, sc, t[0], 100, None)
    mask = torch.ones(100, dtype=torch.bool)
    mask[32:48] = False
    ref, bound = plain.attend_one(q[0], k, v, vs, mask, D ** -0.5, q.dtype)
    plain.assert_within(out[0], ref, bound, "a bad block")
    long = torch.tensor([7 * 16 + 50, 48], dtype=torch.int32)
    t[0, 6] = t[0, 0]
    out, _ = run_attention(ops, q, kc, vc, sc, t, long, "fp8", 5, 0, max_len=7 * 16)
    assert ops.device_diagnostics() & ops.DIAG_DECODE_LEN_CLAMPED


# ------------------------------------------------------------------ the decode step
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D,bs", GEOMETRY)
@pytest.mark.parametrize("window,sinks", [(0, 0), (21, 3)])
def test_decode_step(ops, fmt, dtype, Hq, H, D, bs, window, sinks):
    """Three steps: a row that starts a block, one that joins it, one that grows its scale; codes and
    scales bit for bit, the attention on the updated cache."""
    g = torch.Generator().manual_seed(Hq + D + bs + window)
    lens = [1, bs - 1, bs, 2 * bs + 1, 0, 90]
    kc, vc, sc, t = filled(g, [n + 4 if n else 0 for n in lens], H, D, bs, fmt)
    # the sequences as they stood before: rewrite their first `lens` rows
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    k, v = rows(g, int(cu[-1]), H, D, dtype), rows(g, int(cu[-1]), H, D, dtype)
    plain.write(k, v, kc, vc, sc, t, torch.tensor(lens, dtype=torch.int32), cu, fmt)
    for step in range(3):
        lens = [n + 1 if n else 0 for n in lens]
        ln = torch.tensor(lens, dtype=torch.int32)
        q = rows(g, len(lens), Hq, D, dtype)
        k, v = rows(g, len(lens), H, D, dtype, 4.0 ** step), rows(g, len(lens), H, D, dtype, 4.0 ** step)
        out, dev = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, step=(k, v))
        plain.write(k, v, kc, vc, sc, t, ln, None, fmt)
        for name, a, b in zip(("key codes", "value codes", "scales"), dev, (kc, vc, sc)):
            assert same_bits(a, b), f"step {step}: {name}"
        ref, bound = plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5)
        plain.assert_within(out, ref, bound, f"step {step}")
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("S,Hq,H,D,longest", [
    (9, 8, 8, 128, 3000),     # one workgroup of many waves per sequence and head, several tiles per wave
    (34, 4, 4, 64, 8000),     # three splits
    (17, 12, 12, 64, 8000),   # two splits of small tiles
    (50, 6, 6, 32, 2500),     # two splits of more than 256 workgroups
    (25, 8, 8, 96, 9000),     # none
    (5, 8, 8, 80, 9000)])     # a workgroup per compute unit
@pytest.mark.parametrize("window,sinks", [(0, 0), (1200, 3)])
def test_attention_and_step_launch_shapes(ops, fmt, S, Hq, H, D, longest, window, sinks):
    """The launch is shaped by the longest sequence that may come; the ones that do are ragged, most of
    them with nothing for most of the waves and splits."""
    g = torch.Generator().manual_seed(S + D)
    lens = [int(torch.randint(1, 60, (), generator=g)) for _ in range(S)]
    lens[1], lens[S - 1], lens[2] = 1490, 777, 0
    bs = 16
    kc, vc, sc, t = filled(g, [n + 1 if n else 0 for n in lens], H, D, bs, fmt)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = rows(g, S, Hq, D, torch.bfloat16)
    out, _ = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, max_len=longest)
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5)
    plain.assert_within(out, ref, bound, "attention")
    k, v = rows(g, S, H, D, torch.bfloat16, 3.0), rows(g, S, H, D, torch.bfloat16, 3.0)
    ln = torch.where(ln > 0, ln + 1, ln)
    out, dev = run_attention(ops, q, kc, vc, sc, t, ln, fmt, window, sinks, step=(k, v), max_len=longest)
    plain.write(k, v, kc, vc, sc, t, ln, None, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    ref, bound = plain.decode(q, kc, vc, sc, t, ln, window, sinks, D ** -0.5)
    plain.assert_within(out, ref, bound, "step")
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_decode_step_special_rows(ops, fmt, bs):
    """New rows of zeros, subnormals, infinities, NaN and the largest finite values, starting a block and
    joining one: the codes and scales of the plain write; the outputs of the other sequences."""
    g = torch.Generator().manual_seed(bs)
    H, D = 2, 80
    fills = [0.0, -0.0, 1e-40, 1e-30, 1e4, 3.3e38, float("inf"), float("-inf"), float("nan")]
    S = 2 * len(fills)
    lens = [2 * bs + 1] * len(fills) + [2 * bs + 4] * len(fills)
    kc, vc, sc, t = filled(g, [n - 1 for n in lens], H, D, bs, fmt, spare=S + 5)
    free = [b for b in range(vc.shape[0]) if b not in set(t.flatten().tolist())]
    wide = torch.full((S, 3), -7, dtype=torch.int32)
    wide[:, :t.shape[1]] = t
    wide[:len(fills), 2] = torch.tensor(free[:len(fills)], dtype=torch.int32)
    k, v = rows(g, S, H, D, torch.bfloat16), rows(g, S, H, D, torch.bfloat16)
    for i, f in enumerate(fills + fills):
        k[i, 0, ::7], v[i, 0, 3::5] = f, f
        if i % 2:
            k[i, 1], v[i, 1] = f, f
    q = rows(g, S, 2 * H, D, torch.bfloat16)
    ln = torch.tensor(lens, dtype=torch.int32)
    out, dev = run_attention(ops, q, kc, vc, sc, wide, ln, fmt, 0, 0, step=(k, v))
    plain.write(k, v, kc, vc, sc, wide, ln, None, fmt)
    assert same_bits(dev[2], sc)
    for got, want in zip(dev[:2], (kc, vc)):
        got, want = got.cpu().float(), want.float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    fine = [i for i in range(S) if abs((fills + fills)[i]) < 1e5]
    ref, bound = plain.decode(q[fine], kc, vc, sc, wide[fine], ln[fine], 0, 0, D ** -0.5)
    plain.assert_within(out[fine], ref, bound, "sequences with finite rows")
    ops.check_device_diagnostics()
