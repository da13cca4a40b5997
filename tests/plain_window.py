"""Plain implementations, in 64 bits and on the CPU, of the 8-bit paged cache and of attention with
a sliding window and sink tokens; the bounds of what the kernels' roundings may do to a result."""
import math

import torch

FMAX = {"fp8": 448.0, "int8": 127.0}
CODE_DTYPE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def encode(x, fmt):
    """x f64, already divided by the scale -> codes, to nearest even (f32 holds x exactly here)."""
    x = torch.where(torch.isnan(x), x, x.clamp(-FMAX[fmt], FMAX[fmt]))
    if fmt == "int8":
        return torch.nan_to_num(torch.round(x), nan=0.0).to(torch.int8)
    return x.float().to(torch.float8_e4m3fn)


def need_scale(amax, fmt):
    if amax == 0:
        return 0.0
    k = math.ceil(math.log2(amax / FMAX[fmt]))
    # log2 is rounded: step to the exact answer
    while amax / 2.0 ** k > FMAX[fmt]:
        k += 1
    while amax / 2.0 ** (k - 1) <= FMAX[fmt]:
        k -= 1
    return 2.0 ** max(k, -100)


def k_rows(cache, block):
    """[H, bs, D] codes of one block of a key cache [nb, H, D/16, bs, 16], as f64."""
    b = cache[block]
    return b.permute(0, 2, 1, 3).flatten(2).double()


def v_rows(cache, block):
    return cache[block].transpose(1, 2).double()


def write(key, value, key_cache, value_cache, scales, tables, lens, cu, fmt):
    """In place on CPU tensors, block by block, from the definition."""
    nb, H, D, bs = value_cache.shape
    for s in range(tables.shape[0]):
        r0, r1 = (s, s + 1) if cu is None else (int(cu[s]), int(cu[s + 1]))
        n = int(lens[s])
        if n <= 0 or r1 <= r0 or r1 - r0 > n or n > tables.shape[1] * bs or r1 > key.shape[0]:
            continue
        ctx = n - (r1 - r0)
        for j in range(ctx // bs, (n - 1) // bs + 1):
            b = int(tables[s, j])
            if not 0 <= b < nb:
                continue
            lo, hi = max(ctx, j * bs), min(n, (j + 1) * bs)
            o0 = lo - j * bs
            for which, (rows, cache, get) in enumerate(((key, key_cache, k_rows), (value, value_cache, v_rows))):
                x = rows[r0 + lo - ctx:r0 + hi - ctx].double()               # [m, H, D]
                codes = get(cache, b)                                          # [H, bs, D]
                new = cache[b].clone()
                for h in range(H):
                    xh = x[:, h]
                    finite = xh[torch.isfinite(xh)].abs()
                    old = float(scales[b, h, which]) if o0 else 0.0
                    sc = max(old, need_scale(float(finite.max()) if finite.numel() else 0.0, fmt))
                    if old > 0 and sc > old:
                        put(new, h, 0, encode(codes[h, :o0] * (old / sc), fmt), which)
                    put(new, h, o0, encode(xh / (sc or 1.0), fmt), which)
                    scales[b, h, which] = sc
                cache[b] = new


def put(block, h, off, codes, which):
    """codes [m, D] into slots off .. of one head of a block in the cache's layout."""
    m, D = codes.shape
    raw = block.view(torch.uint8) if block.dtype != torch.int8 else block
    codes = codes.view(torch.uint8) if block.dtype != torch.int8 else codes
    if which == 0:
        raw[h, :, off:off + m, :] = codes.reshape(m, D // 16, 16).transpose(0, 1)
    else:
        raw[h, :, off:off + m] = codes.T


def gather(cache_k, cache_v, scales, table, n, x):
    """K and V [H, n, D] of a sequence in f64, the block of every token, and the V codes."""
    nb, H, D, bs = cache_v.shape
    ids = [int(b) for b in table[:-(-n // bs)]]
    k = torch.cat([cache_k[b].permute(0, 2, 1, 3).flatten(2).double() for b in ids], 1)[:, :n]
    v = torch.cat([v_rows(cache_v, b) for b in ids], 1)[:, :n]
    if scales is None:
        return k, v, torch.ones(H, n, dtype=torch.float64)
    ks = torch.stack([scales[b, :, 0] for b in ids], 1).double().repeat_interleave(bs, 1)[:, :n]
    vs = torch.stack([scales[b, :, 1] for b in ids], 1).double().repeat_interleave(bs, 1)[:, :n]
    return k * ks[..., None], v * vs[..., None], vs


def visible(n, window, sinks):
    j = torch.arange(n)
    return (j >= 0) if window == 0 else (j >= n - window) | (j < sinks)


def attend_one(q, k, v, vs, mask, scale, dtype):
    """q [Hq, D], k/v [H, n, D], mask [n]; returns (out, bound) f64 [Hq, D].

    The bound follows the kernels' arithmetic, u = half a step of `dtype`:
      * the weights are rounded once to `dtype` (u of each, or - f16 - half a subnormal step
        2^-25 of the largest weight, V's scale included), the result once (u);
      * scores are f32 sums of D products and two scalings: (D + 4) 2^-24 of sum |q k|, which moves
        a weight, and through numerator and denominator the result, by at most twice that;
      * exp2 to 2^-22 of its value (twice: weight and rescaling), sums of n weights to n 2^-24;
      * a weight below 2^-126, f32's smallest normal number, may come out as 0 (as p, as p times V's
        scale, or when it is rescaled): 2^-126 per weight in front of |v| and of |code|, |v| = |code|
        * scale.  (It is all there is where the heavy tokens have code 0: sum p v = 1e-40.)"""
    H, n, D = k.shape
    group = q.shape[0] // H
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    u = HALF_STEP[dtype]
    if not bool(mask.any()):
        return out, bound
    for h in range(q.shape[0]):
        kv = h // group
        kk, vv, ss = k[kv][mask], v[kv][mask], vs[kv][mask]
        s = (kk @ q[h].double()) * scale
        size = (kk.abs() @ q[h].double().abs()) * abs(scale)
        p = torch.exp(s - s.max())
        l = p.sum()
        out[h] = (p @ vv) / l
        spread = (p @ vv.abs()) / l
        rel = u + 2 * float(size.max()) * (D + 4) * 2.0 ** -24 + 4 * 2.0 ** -22 + 2 * len(p) * 2.0 ** -24
        bound[h] = spread * rel + out[h].abs() * u
        code = torch.where(ss > 0, 1 / ss, torch.zeros_like(ss))[:, None] * vv.abs()
        bound[h] += 2.0 ** -126 * (2 * vv.abs() + code).sum(0) / l
        if dtype == torch.float16:
            bound[h] += 2.0 ** -25 * float((p * ss).max()) * code.sum(0) / l + 2.0 ** -25
    return out, bound


def decode(q, cache_k, cache_v, scales, tables, lens, window, sinks, scale):
    outs, bounds = [], []
    H, D = cache_v.shape[1], cache_v.shape[2]
    for s in range(q.shape[0]):
        n = int(lens[s])
        if n <= 0:
            z = torch.zeros(q.shape[1], D, dtype=torch.float64)
            outs.append(z), bounds.append(z)
            continue
        k, v, vs = gather(cache_k, cache_v, scales, tables[s], n, None)
        o, b = attend_one(q[s].cpu(), k, v, vs, visible(n, window, sinks), scale, q.dtype)
        outs.append(o), bounds.append(b)
    return torch.stack(outs), torch.stack(bounds)


def assert_within(got, ref, bound, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = (got - ref).abs() - bound
    worst = float(excess.max()) if excess.numel() else 0.0
    assert worst <= 0, f"{what}: off by {float((got - ref).abs().max()):.3e}, {worst:.3e} over the bound"
