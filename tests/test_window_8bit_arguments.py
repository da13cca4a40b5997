"""Refusals of the 8-bit cache and the windowed attention, without a GPU: the operators check their
arguments before they look for a device, the C entry points before they touch one."""
import pytest
import torch

import vllm_paged_compression_amd.ops as ops
from vllm_paged_compression_amd import _lib

P = 1 << 20   # stands for an aligned device pointer; nothing dereferences it


def cache(nb=6, H=2, D=64, bs=16, dtype=torch.int8):
    return (torch.zeros(nb, H, D // 16, bs, 16, dtype=dtype), torch.zeros(nb, H, D, bs, dtype=dtype),
            torch.zeros(nb, H, 2))


def tables(S=3, M=2):
    return torch.zeros(S, M, dtype=torch.int32), torch.ones(S, dtype=torch.int32)


def rows(n=3, H=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(n, H, D, dtype=dtype)


def refused(match, fn, *args, error=RuntimeError):
    with pytest.raises(error, match=match):
        fn(*args)


def test_good_arguments_reach_the_device_check():
    kc, vc, sc = cache()
    t, ln = tables()
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    q = rows(3, 4)
    for call in (lambda: ops.reshape_and_cache_8bit(rows(), rows(), kc, vc, sc, t, ln, cu, 1, "int8"),
                 lambda: ops.reshape_and_cache_8bit(rows(), rows(), kc, vc, sc, t, ln, None, 1, "int8"),
                 lambda: ops.paged_attention_8bit(q.clone(), q, kc, vc, sc, 2, 0.1, t, ln, 16, 32, "int8", 5, 1),
                 lambda: ops.decode_step_8bit(q.clone(), q, rows(), rows(), kc, vc, sc, 2, 0.1, t, ln, 16, 32, "int8"),
                 lambda: ops.paged_attention_window(q.clone(), q, torch.zeros(6, 2, 8, 16, 8, dtype=q.dtype),
                                                    torch.zeros(6, 2, 64, 16, dtype=q.dtype), 2, 0.1, t, ln, 16, 32, 5),
                 lambda: ops.prefill_window(q, rows(), rows(), cu, cu, 1, 0.1, 5, 1)):
        with pytest.raises(RuntimeError, match="run on the GPU only"):
            call()


def test_8bit_write_refusals():
    kc, vc, sc = cache()
    t, ln = tables()
    good = [rows(), rows(), kc, vc, sc, t, ln, None, 1, "int8"]

    def bad(match, error=RuntimeError, **kw):
        names = ["key", "value", "key_cache", "value_cache", "kv_scales", "block_tables", "seq_lens", "cu_q",
                 "max_q_len", "kv_cache_dtype"]
        refused(match, ops.reshape_and_cache_8bit, *[kw.get(n, g) for n, g in zip(names, good)], error=error)

    bad("kv_cache_dtype must be", ValueError, kv_cache_dtype="auto")
    bad("is held in", kv_cache_dtype="fp8")
    bad("is held in", key_cache=kc.view(torch.uint8), value_cache=vc.view(torch.uint8))
    bad("differ in dtype", value_cache=vc.view(torch.uint8))
    bad("bfloat16 or float16 rows", key=rows(dtype=torch.float32), value=rows(dtype=torch.float32))
    bad("key_cache must be", key_cache=kc.transpose(2, 3))
    bad("5-d", key_cache=vc)
    bad("contiguous", value_cache=torch.zeros(6, 2, 64, 32, dtype=torch.int8)[..., ::2])
    bad("kv_scales", kv_scales=sc[:, :, :1])
    bad("kv_scales", kv_scales=sc.double())
    bad("int32", block_tables=t.long())
    bad("block_tables must be", block_tables=torch.zeros(3, 4, dtype=torch.int32)[:, ::2])
    bad("seq_lens must be", seq_lens=ln[:2])
    bad("one row per sequence", key=rows(4), value=rows(4))
    bad("cu_q", cu_q=torch.zeros(3, dtype=torch.int32))
    bad("cu_q", cu_q=torch.zeros(4, dtype=torch.int64))
    bad("negative max_q_len", ValueError, max_q_len=-1)
    bad("key must be", key=rows(H=3))
    bad("value must be", value=rows(D=32))
    bad("differ in shape or dtype", value=rows(dtype=torch.float16))
    bad("must be dense", key=torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2])
    bad("16-byte aligned", key=torch.zeros(3 * 2 * 64 + 1, dtype=torch.bfloat16)[1:].view(3, 2, 64))
    bad("16-byte aligned", key=torch.zeros(3, 2 * 64 + 1, dtype=torch.bfloat16)[:, :128].unflatten(1, (2, 64)))


def test_8bit_attention_and_step_refusals():
    kc, vc, sc = cache()
    t, ln = tables()
    q = rows(3, 4)
    att = lambda **kw: ops.paged_attention_8bit(  # noqa: E731
        kw.get("out", q.clone()), kw.get("q", q), kc, vc, sc, kw.get("H", 2), 0.1, t, ln, kw.get("bs", 16), 32, "int8",
        kw.get("window", 0), kw.get("sinks", 0))
    refused("num_kv_heads/block_size", lambda: att(H=4))
    refused("num_kv_heads/block_size", lambda: att(bs=8))
    refused("multiple", lambda: att(q=rows(3, 3)))
    refused("query must be", lambda: att(q=rows(2, 4)))
    refused("query must be", lambda: att(q=rows(3, 4, 32)))
    refused("out must be", lambda: att(out=q.clone().half()))
    refused("out must be", lambda: att(out=torch.zeros(3, 8, 64, dtype=q.dtype)[:, ::2]))
    refused("negative", lambda: att(window=-1), error=ValueError)
    refused("negative", lambda: att(sinks=-1), error=ValueError)
    step = lambda k, v: ops.decode_step_8bit(q.clone(), q, k, v, kc, vc, sc, 2, 0.1, t, ln, 16, 32, "int8")  # noqa: E731
    refused("of query's dtype", lambda: step(rows(dtype=torch.float16), rows(dtype=torch.float16)))
    refused("of query's dtype", lambda: step(rows(4), rows(4)))
    refused("differ in shape", lambda: step(rows(), rows(4)))


def test_window_refusals():
    t, ln = tables()
    q, kc, vc = rows(3, 4), torch.zeros(6, 2, 8, 16, 8, dtype=torch.bfloat16), torch.zeros(6, 2, 64, 16, dtype=torch.bfloat16)
    refused("share bfloat16 or float16", ops.paged_attention_window, q, q, kc.half(), vc.half(), 2, 0.1, t, ln, 16, 32, 4)
    refused("share bfloat16 or float16", ops.paged_attention_window, q.float(), q.float(), kc.float(), vc.float(), 2, 0.1, t, ln, 16, 32, 4)
    refused("negative", ops.paged_attention_window, q.clone(), q, kc, vc, 2, 0.1, t, ln, 16, 32, -4, error=ValueError)
    cu = torch.tensor([0, 3], dtype=torch.int32)
    pf = lambda **kw: ops.prefill_window(  # noqa: E731
        kw.get("q", q), kw.get("k", rows()), kw.get("v", rows()), kw.get("cu", cu), kw.get("cu2", cu), 3, 0.1,
        kw.get("window", 2), kw.get("sinks", 0), kw.get("out"))
    refused("multiple of Hkv", lambda: pf(q=rows(3, 5)))
    refused("expected", lambda: pf(v=rows(4)))
    refused("key must be", lambda: pf(k=rows(D=32), v=rows(D=32)))
    refused("share", lambda: pf(v=rows(dtype=torch.float16)))
    refused("cu_q/cu_kv", lambda: pf(cu2=torch.zeros(3, dtype=torch.int32)))
    refused("cu_q/cu_kv", lambda: pf(cu=cu.long(), cu2=cu.long()))
    refused("negative", lambda: pf(window=-1), error=ValueError)
    refused("negative", lambda: pf(sinks=-1), error=ValueError)
    refused("out must have", lambda: pf(out=q.half()))


def said(lib, rc, code, text):
    assert rc == code and text in lib.pe_last_error(), (rc, lib.pe_last_error())


def test_c_entry_points_refuse_before_the_device():
    lib = _lib.load()

    def write(H=2, D=64, bs=16, nb=6, M=2, stride=64, kv=2048, dtype=2, fmt=2, key=P, S=3, T=3, n=1, cu=None):
        return lib.pe_reshape_and_cache_8bit(key, P, P, P, P, P, P, cu, S, T, n, stride, stride, H, D, bs, nb, M,
                                             kv, D * bs, dtype, fmt, None)
    assert write(S=0) == 0 and write(T=0) == 0 and write(n=0) == 0
    said(lib, write(S=-1), 1, b"negative")
    said(lib, write(key=None), 1, b"null pointer")
    said(lib, write(fmt=0), 2, b"kv_format")
    said(lib, write(dtype=0), 2, b"dtype")
    said(lib, write(D=120), 2, b"head size")
    said(lib, write(bs=64), 2, b"block size")
    said(lib, write(M=1 << 27), 2, b"2^30")
    said(lib, write(kv=2056), 1, b"16-byte")
    said(lib, write(stride=65), 1, b"16-byte")
    said(lib, write(T=2), 1, b"one row per sequence")
    said(lib, write(S=70000, T=70000), 2, b"grid")

    def attend(Hq=4, H=2, D=64, bs=16, M=2, q=P, scales=P, window=0, sinks=0, S=3, dtype=2, fmt=1, stride=256):
        return lib.pe_paged_decode_8bit(P, q, P, P, scales, P, P, S, Hq, H, D, bs, 6, M, stride, 2048, 1024, 0.1, 32,
                                        window, sinks, dtype, fmt, None, 0, None)
    assert attend(S=0) == 0
    said(lib, attend(scales=None), 1, b"null pointer")
    said(lib, attend(q=None), 1, b"null pointer")
    said(lib, attend(window=-1), 1, b"negative")
    said(lib, attend(Hq=5), 1, b"multiple")
    said(lib, attend(q=P + 2), 1, b"16-byte")
    said(lib, attend(stride=257), 1, b"16-byte")
    said(lib, attend(D=100), 2, b"head size")

    def window(D=64, bs=16, M=2, dtype=2, w=4, s=0, cachep=P):
        return lib.pe_paged_decode_window(P, P, cachep, P, P, P, 3, 4, 2, D, bs, 6, M, 256, 2048, 1024, 0.1, 32, w, s,
                                          dtype, None, 0, None)
    said(lib, window(dtype=0), 2, b"dtype")
    said(lib, window(s=-1), 1, b"negative")
    said(lib, window(cachep=P + 8), 1, b"16-byte")
    said(lib, window(D=72), 2, b"head size")
    said(lib, window(bs=4), 2, b"block size")

    def prefill(D=64, scale=0.1, dtype=2, w=4, n=10, stride=256, S=1):
        return lib.pe_prefill_window(P, P, P, P, P, P, S, n, 99, 99, 4, 2, D, stride, stride, stride, stride, scale, w, 0, dtype, None)
    assert prefill(S=0) == 0 and prefill(n=0) == 0
    said(lib, prefill(D=72), 2, b"head size")
    said(lib, prefill(scale=0.0), 2, b"scale")
    said(lib, prefill(scale=float("nan")), 2, b"scale")
    said(lib, prefill(scale=float("inf")), 2, b"scale")
    said(lib, prefill(dtype=0), 2, b"dtype")
    said(lib, prefill(w=-1), 1, b"negative")
    said(lib, prefill(stride=1 << 24), 1, b"2^24")
    said(lib, prefill(stride=260 + 2), 1, b"16-byte")
    rc = lib.pe_decode_step_8bit(P, P, None, P, P, P, P, P, P, 3, 4, 2, 64, 16, 6, 2, 256, 128, 128, 2048, 1024, 0.1,
                                 32, 0, 0, 2, 2, None, 0, None)
    said(lib, rc, 1, b"null pointer")


def test_workspace_size_is_a_host_function():
    lib = _lib.load()
    size = lambda S, n, w=0, s=0: lib.pe_paged_window_workspace_bytes(S, 32, 8, 128, n, w, s, 1)  # noqa: E731
    assert size(0, 1000) == 0 and size(64, 0) == 0
    assert size(1, 100000) >= size(1, 100000, 256, 4)      # a window reads less, and splits less
    assert size(4, 2 ** 31 - 1) >= 0
