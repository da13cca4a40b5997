"""The 8-bit cache and the windowed attention as a server uses them together: prompt, write, steps with
pages given away and taken again, eviction, forked pages, replayed graphs, several streams."""
import pytest
import torch

import plain_window as plain
from test_gpu_8bit_cache import FORMATS, filled, garbage_cache, rows, same_bits
from test_gpu_window import prefill_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import vllm_paged_compression_amd as pkg
    import vllm_paged_compression_amd.ops as ops
    pkg.load_library()
    return ops


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_windowed_generation(ops, fmt, bs):
    """Two prompts through a window, their rows into 8-bit pages, 40 steps.  A page that leaves the
    window goes back to the pool and is handed out again with what it held."""
    g = torch.Generator().manual_seed(bs)
    Hq, H, D, W, sinks, dtype = 8, 2, 64, 50, 4, torch.bfloat16
    lens, scale = [133, 70], D ** -0.5
    T = sum(lens)
    q, k, v = rows(g, T, Hq, D, dtype), rows(g, T, H, D, dtype), rows(g, T, H, D, dtype)
    cu = torch.tensor([0, lens[0], T], dtype=torch.int32)
    out = ops.prefill_window(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), cu.cuda(), max(lens), scale, W, sinks)
    plain.assert_within(out, *prefill_reference(q, k, v, lens, lens, W, sinks, scale), "prompt")

    width = -(-(max(lens) + 40) // bs)
    nb = sum(-(-n // bs) for n in lens) + 3        # too few pages without recycling (bs <= 16)
    kc, vc, sc = garbage_cache(g, nb, H, D, bs, fmt)
    free = torch.randperm(nb, generator=g).tolist()
    t = torch.full((2, width), -1, dtype=torch.int32)
    for s, n in enumerate(lens):
        for j in range(-(-n // bs)):
            t[s, j] = free.pop()
    dev = [x.cuda() for x in (kc, vc, sc)]
    ln = torch.tensor(lens, dtype=torch.int32)
    plain.write(k, v, kc, vc, sc, t, ln, cu, fmt)
    ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), *dev, t.cuda(), ln.cuda(), cu.cuda(), max(lens), fmt)
    for step in range(40):
        for s in range(2):
            lens[s] += 1
            j = (lens[s] - 1) // bs
            for old in range(j):                   # pages without a visible token
                if t[s, old] >= 0 and old * bs >= sinks and (old + 1) * bs <= lens[s] - W:
                    free.append(int(t[s, old]))
                    t[s, old] = -1
            if t[s, j] < 0:
                t[s, j] = free.pop()
        ln = torch.tensor(lens, dtype=torch.int32)
        q, k, v = (rows(g, 2, h, D, dtype, 1.05 ** step) for h in (Hq, H, H))
        out = torch.full_like(q, float("nan")).cuda()
        ops.decode_step_8bit(out, q.cuda(), k.cuda(), v.cuda(), *dev, H, scale, t.cuda(), ln.cuda(), bs,
                             width * bs, fmt, W, sinks)
        plain.write(k, v, kc, vc, sc, t, ln, None, fmt)
        assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc))), f"step {step}"
        known = t.clamp(min=0)                     # the plain gather reads every page; hidden ones do not count
        zk, zv, zs = torch.nan_to_num(kc.float()).to(kc.dtype), torch.nan_to_num(vc.float()).to(vc.dtype), torch.nan_to_num(sc, nan=0.0, posinf=0.0)
        ref, bound = plain.decode(q, zk, zv, zs, known, ln, W, sinks, scale)
        plain.assert_within(out, ref, bound, f"step {step}")
    ops.check_device_diagnostics()


@pytest.mark.parametrize("fmt", FORMATS)
def test_eviction_on_8bit_pages(ops, fmt):
    """streamingLLM's decision works on tables alone: the compacted table read by the 8-bit attention."""
    g = torch.Generator().manual_seed(3)
    H, D, bs, budget = 2, 128, 16, 128
    lens = [budget + bs] * 3       # the decision falls on a block boundary past the budget
    kc, vc, sc, t = filled(g, lens, H, D, bs, fmt)
    M = t.shape[1]
    dev = [x.cuda() for x in (kc, vc, sc)]
    rmv, small, _ = ops.evict_select_compact(t.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                             torch.full((3,), M, dtype=torch.int32).cuda(), "streamingLLM", budget, bs,
                                             out_width=M)
    rmv = rmv.cpu().tolist()
    assert min(rmv) >= 0
    kept = torch.stack([torch.cat([t[s, :r], t[s, r + 1:]]) for s, r in enumerate(rmv)])
    assert torch.equal(small.cpu()[:, :M - 1], kept)
    ln = torch.tensor(lens, dtype=torch.int32) - bs
    q = rows(g, 3, 8, D, torch.float16)
    out = torch.empty_like(q).cuda()
    ops.paged_attention_8bit(out, q.cuda(), *dev, H, D ** -0.5, small, ln.cuda(), bs, int(ln.max()), fmt)
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, kept, ln, 0, 0, D ** -0.5))


def test_forked_pages(ops):
    """A forked sequence shares the full pages and gets a copy of the last one, codes and scales
    (swap_blocks moves bytes); parent and child then grow apart."""
    g = torch.Generator().manual_seed(4)
    H, D, bs, fmt = 2, 64, 16, "fp8"
    kc, vc, sc, t = filled(g, [40], H, D, bs, fmt)
    own = [b for b in range(vc.shape[0]) if b not in t[0].tolist()][0]
    pair = torch.tensor([[int(t[0, 2]), own]])
    dev = [x.cuda() for x in (kc, vc, sc)]
    for x in dev:
        ops.swap_blocks(x, x, pair)
    for x in (kc, vc, sc):
        x[own] = x[pair[0, 0]]
    two = torch.cat([t, t])
    two[1, 2] = own
    ln = torch.tensor([41, 41], dtype=torch.int32)
    k, v, q = rows(g, 2, H, D, torch.bfloat16, 9.0), rows(g, 2, H, D, torch.bfloat16, 9.0), rows(g, 2, 4, D, torch.bfloat16)
    out = torch.empty_like(q).cuda()
    ops.decode_step_8bit(out, q.cuda(), k.cuda(), v.cuda(), *dev, H, D ** -0.5, two.cuda(), ln.cuda(), bs, 48, fmt)
    plain.write(k, v, kc, vc, sc, two, ln, None, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    plain.assert_within(out, *plain.decode(q, kc, vc, sc, two, ln, 0, 0, D ** -0.5))


@pytest.mark.parametrize("seqs,length", [(2, 60), (1, 3000)])
def test_replayed_steps(ops, seqs, length):
    """One captured step (one launch, and attention + merge for the long sequence) replayed with the
    length advanced on the device and eager work between the replays; every replay against eager."""
    g = torch.Generator().manual_seed(5)
    Hq, H, D, bs, fmt, steps = 8, 2, 128, 16, "fp8", 6
    kc, vc, sc, t = filled(g, [length + steps] * seqs, H, D, bs, fmt)
    start = torch.full((seqs,), length, dtype=torch.int32).cuda()
    # the sequences as they stood before the steps: their rows again, up to `length`
    cu = (torch.arange(seqs + 1) * length).to(torch.int32).cuda()
    kk, vv = (rows(g, seqs * length, H, D, torch.bfloat16).cuda() for _ in range(2))
    a = [x.cuda() for x in (kc, vc, sc)]
    td = t.cuda()
    ops.reshape_and_cache_8bit(kk, vv, *a, td, start, cu, length, fmt)
    b = [x.clone() for x in a]
    q, k, v = (torch.empty(seqs, h, D, dtype=torch.bfloat16, device="cuda") for h in (Hq, H, H))
    feed = [[rows(g, seqs, h, D, torch.bfloat16, 2.0 ** s).cuda() for h in (Hq, H, H)] for s in range(steps)]
    ln, out = start.clone(), torch.empty_like(q)
    for buf, x in zip((q, k, v), feed[0]):
        buf.copy_(x)

    def step(caches):
        ops.decode_step_8bit(out, q, k, v, *caches, H, D ** -0.5, td, ln, bs, t.shape[1] * bs, fmt)

    warm = [x.clone() for x in a]
    ln += 1
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    ln.copy_(start)
    for s in range(steps):
        for buf, x in zip((q, k, v), feed[s]):
            buf.copy_(x)
        ln += 1
        out.fill_(float("nan"))
        graph.replay()
        got = out.clone()
        step(b)                                    # eager, the same step on the other cache
        assert torch.equal(got, out), f"replay {s}"
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b)), f"replay {s}"
        torch.cuda.synchronize()


def test_two_graphs_and_two_streams_do_not_share(ops):
    """Split launches: two graphs replayed at once on two streams, and eager calls beside them, give what
    each gives alone (their partials lie in buffers of their own)."""
    g = torch.Generator().manual_seed(6)
    H, D, bs, fmt, n = 1, 128, 16, "int8", 6000
    kc, vc, sc, t = filled(g, [n], H, D, bs, fmt)
    dev = [x.cuda() for x in (kc, vc, sc)]
    td = t.cuda()
    ln = torch.tensor([n], dtype=torch.int32).cuda()
    qs = [rows(g, 1, 4, D, torch.bfloat16).cuda() for _ in range(3)]
    outs = [torch.empty_like(q) for q in qs]

    def call(i):
        ops.paged_attention_8bit(outs[i], qs[i], *dev, H, D ** -0.5, td, ln, bs, n, fmt)

    alone = []
    for i in range(3):
        call(i)
        alone.append(outs[i].clone())
    graphs, streams = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            for _ in range(20):
                call(i)
    for rep in range(5):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(20):
                call(2)
        torch.cuda.synchronize()
        for i in range(3):
            assert torch.equal(outs[i], alone[i]), f"repetition {rep}, call {i}"


def test_same_call_twice_gives_the_same_bits(ops):
    g = torch.Generator().manual_seed(7)
    kc, vc, sc, t = filled(g, [2500, 900], 2, 64, 8, "fp8")
    dev = [x.cuda() for x in (kc, vc, sc)]
    ln, td = torch.tensor([2500, 900], dtype=torch.int32).cuda(), t.cuda()
    q = rows(g, 2, 8, 64, torch.float16).cuda()
    got = []
    for _ in range(3):
        out = torch.empty_like(q)
        ops.paged_attention_8bit(out, q, *dev, 2, 0.1, td, ln, 8, 2500, "fp8", 1000, 7)
        got.append(out)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    lens = [700, 90]
    cu = torch.tensor([0, 700, 790], dtype=torch.int32).cuda()
    x = [rows(g, 790, h, 64, torch.bfloat16).cuda() for h in (8, 2, 2)]
    a, b = (ops.prefill_window(*x, cu, cu, max(lens), 0.125, 100, 3) for _ in range(2))
    assert torch.equal(a, b)


def test_padded_batch_rows(ops):
    """Rows of a padded batch (length 0, any table, any row in key/value): zeros out, nothing written."""
    g = torch.Generator().manual_seed(8)
    H, D, bs, fmt = 2, 64, 16, "int8"
    kc, vc, sc, t = filled(g, [30], H, D, bs, fmt)
    t = torch.cat([t, t, torch.full_like(t, 2 ** 31 - 1)])
    ln = torch.tensor([31, 0, 0], dtype=torch.int32)
    q, k, v = (rows(g, 3, h, D, torch.bfloat16) for h in (4, H, H))
    k[1:] = float("nan")
    dev = [x.cuda() for x in (kc, vc, sc)]
    out = torch.full_like(q, float("nan")).cuda()
    ops.device_diagnostics()
    ops.decode_step_8bit(out, q.cuda(), k.cuda(), v.cuda(), *dev, H, 0.1, t.cuda(), ln.cuda(), bs, 32, fmt)
    plain.write(k, v, kc, vc, sc, t, ln, None, fmt)
    assert all(same_bits(a, b) for a, b in zip(dev, (kc, vc, sc)))
    assert (out[1:] == 0).all() and torch.isfinite(out[0]).all()
    assert ops.device_diagnostics() == 0
    # a length that the table cannot hold: reported, cut for the attention, not written
    before = [x.clone() for x in dev]
    ln = torch.tensor([33, 0, 0], dtype=torch.int32)
    ops.decode_step_8bit(out, q.cuda(), k.cuda(), v.cuda(), *dev, H, 0.1, t.cuda(), ln.cuda(), bs, 32, fmt)
    assert ops.device_diagnostics() == ops.DIAG_DECODE_LEN_CLAMPED | ops.DIAG_APPEND_MISMATCH
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(dev, before))


def test_offsets_past_32_bits(ops):
    """A pool of more than 4 GiB: the last pages are written and read."""
    H, D, bs, fmt, nb = 8, 256, 32, "int8", 70000          # 64 KiB per page and tensor: 4.6 GB each
    g = torch.Generator().manual_seed(9)
    kc = torch.zeros(nb, H, D // 16, bs, 16, dtype=torch.int8, device="cuda")
    vc = torch.zeros(nb, H, D, bs, dtype=torch.int8, device="cuda")
    sc = torch.zeros(nb, H, 2, device="cuda")
    t = torch.tensor([[nb - 1, 65537]], dtype=torch.int32)
    n = 50
    k, v, q = rows(g, n, H, D, torch.bfloat16), rows(g, n, H, D, torch.bfloat16), rows(g, 1, 2 * H, D, torch.bfloat16)
    ln, cu = torch.tensor([n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    ops.reshape_and_cache_8bit(k.cuda(), v.cuda(), kc, vc, sc, t.cuda(), ln.cuda(), cu.cuda(), n, fmt)
    out = torch.empty_like(q).cuda()
    ops.paged_attention_8bit(out, q.cuda(), kc, vc, sc, H, D ** -0.5, t.cuda(), ln.cuda(), bs, n, fmt)
    ids = t[0].long()
    small = [x[ids.cuda()].cpu() for x in (kc, vc, sc)]
    want = [torch.zeros_like(x) for x in small]
    local = torch.tensor([[0, 1]], dtype=torch.int32)
    plain.write(k, v, *want, local, ln, cu, fmt)
    assert all(torch.equal(a, b) for a, b in zip(small, want))
    assert int(kc.count_nonzero()) == int(small[0].count_nonzero())
    plain.assert_within(out, *plain.decode(q, *want, local, ln, 0, 0, D ** -0.5))
    step = [rows(g, 1, h, D, torch.bfloat16) for h in (H, H)]
    ln = ln + 1
    ops.decode_step_8bit(out, q.cuda(), step[0].cuda(), step[1].cuda(), kc, vc, sc, H, D ** -0.5, t.cuda(), ln.cuda(), bs, n + 1, fmt)
    plain.write(*step, *want, local, ln, None, fmt)
    assert all(torch.equal(x[ids.cuda()].cpu(), b) for x, b in zip((kc, vc, sc), want))
