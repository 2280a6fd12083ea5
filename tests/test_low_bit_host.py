"""Host side of the low-bit serving operators, without a GPU: refusals of the C interface before any launch, of the Python
layer, shapes on meta tensors, and the float64 restatements against values worked out by hand."""
import inspect

import pytest
import torch

import helion_amd as hx
from helion_amd import _lib
from oracle import low_bit as ref

A = 1 << 20  # an aligned address that is never followed


def test_norm_and_quantize_refusals():
    lib = _lib.load()
    norm = lambda **k: lib.hx_rms_norm_int8(*[{**dict(x=A, xs=8, r=None, rs=0, w=A, eps=1e-6, h=None, q=A, s=A, rows=2, width=8, dt=1), **k}[n]
                                              for n in ("x", "xs", "r", "rs", "w", "eps", "h", "q", "s", "rows", "width", "dt")], None)
    assert norm(rows=-1) == -1 and b"negative" in lib.hx_last_error()
    assert norm(rows=0) == 0
    assert norm(dt=3) == -1
    assert norm(width=0) == -2 and norm(width=65537, xs=65537) == -2
    assert norm(x=None) == -1 and norm(w=None) == -1 and norm(q=None) == -1 and norm(s=None) == -1
    assert norm(r=A, rs=8) == -1                       # a residual without somewhere to put the sum
    assert norm(xs=7) == -1 and norm(r=A, rs=7, h=A) == -1
    assert norm(x=A + 1) == -2 and norm(s=A + 2) == -2 and norm(dt=2, x=A + 2) == -2
    assert lib.hx_int8_quantize_per_token(A, 8, A, A, 1 << 31, 8, 1, None) == -2
    assert lib.hx_int8_quantize_per_token(None, 8, A, A, 2, 8, 1, None) == -1


def test_int8_gemm_refusals_and_workspace():
    lib = _lib.load()
    base = dict(a=A, b=A, c=A, M=4, N=4, K=128, lda=128, bk=1, bn=128, ldc=4, sa=A, sb=A, bias=None, bdt=0, dt=1, ws=None, wsb=0)
    gemm = lambda **k: lib.hx_int8_gemm(*{**base, **k}.values(), None)
    assert gemm(M=-1) == -1 and gemm(M=0) == 0 and gemm(N=0) == 0
    assert gemm(dt=3) == -1 and gemm(bias=A, bdt=3) == -1
    assert gemm(K=131072, lda=131072, bn=131072) == -2 and b"131071" in lib.hx_last_error()
    assert gemm(K=0) == -2
    assert gemm(a=None) == -1 and gemm(b=None) == -1 and gemm(c=None) == -1 and gemm(sa=None) == -1 and gemm(sb=None) == -1
    assert gemm(lda=127) == -1 and gemm(ldc=3) == -1 and gemm(bk=0) == -1
    assert gemm(c=A + 1) == -2 and gemm(sa=A + 2) == -2 and gemm(bias=A + 1) == -2
    assert gemm(M=1 << 31, lda=128) == -2 and gemm(M=1 << 26) == -2                # 4 GB and more of operand
    assert gemm(bk=4, bn=1) == -3 and b"workspace" in lib.hx_last_error()           # another stride order: copied
    need = lambda m, n, k, lda, bk, bn, a=A, b=A: lib.hx_int8_gemm_workspace_bytes(m, n, k, lda, bk, bn, a, b)
    assert need(300, 300, 256, 256, 1, 256) == 0
    assert need(300, 300, 272, 272, 1, 272) == 0                                     # both read in place and behind k
    assert need(300, 300, 272, 272, 1, 272, A + 1) == 300 * 384 + (-300 * 384) % 256 # a copied, b read in place
    assert need(300, 300, 256, 256, 1, 256, A + 1) == 300 * 256 and need(300, 300, 256, 256, 1, 256, A, A + 8) == 300 * 256
    assert need(300, 300, 100, 100, 1, 100) == 2 * 300 * 128 + 2 * (-300 * 128 % 256)
    assert need(0, 4, 4, 4, 1, 4) == 0 and need(4, 4, 200000, 200000, 1, 200000) == 0


def test_kv4_refusals():
    lib = _lib.load()
    wb = dict(k=A, v=A, kc=A, ks=A, vc=A, vs=A, slots=A, wide=1, tokens=4, heads=2, D=128, pages=3, page=16, kt=256, kh=128, vt=256, vh=128, dt=1)
    write = lambda **k: lib.hx_kv4_write(*{**wb, **k}.values(), None)
    assert write(tokens=-1) == -1 and write(pages=-1) == -1 and write(heads=-1) == -1
    assert write(tokens=0) == 0 and write(pages=0, kc=None, ks=None, vc=None, vs=None) == 0
    assert write(page=24) == -2 and write(page=8) == -2 and write(page=2048) == -2
    assert write(D=96) == -2 and write(dt=3) == -1
    assert write(kc=None) == -1 and write(slots=None) == -1 and write(k=None) == -1
    assert write(vs=A + 8) == -2 and write(slots=A + 4) == -2 and write(k=A + 1) == -2
    rb = dict(kc=A, ks=A, vc=A, vs=A, slots=A, wide=0, k=A, v=A, tokens=4, heads=2, D=64, pages=3, page=32, dt=0)
    read = lambda **k: lib.hx_kv4_read(*{**rb, **k}.values(), None)
    assert read(tokens=-2) == -1 and read(dt=9) == -1 and read(v=None) == -1 and read(k=A + 8) == -2 and read(D=32) == -2
    ab = dict(q=A, qt=256, qh=128, kc=A, ks=A, vc=A, vs=A, table=A, ts=4, lens=A, start=None, out=A, tokens=2, batch=2, heads=2, kv=1, D=128,
              pages=8, page=16, width=4, mq=1, scale=0.1, causal=1, dt=1, ws=None, wsb=0)
    att = lambda **k: lib.hx_kv4_attention(*{**ab, **k}.values(), None)
    assert att(tokens=-1) == -1 and att(width=-1) == -1 and att(mq=-1) == -1
    assert att(heads=3, kv=2) == -1 and att(kv=0) == -1
    assert att(tokens=3) == -1 and b"query_start" in lib.hx_last_error()
    assert att(ts=3) == -1 and att(lens=None) == -1 and att(table=None) == -1 and att(q=None) == -1
    assert att(out=A + 8) == -2 and att(q=A + 1) == -2 and att(lens=A + 2) == -2
    assert att(dt=3) == -1 and att(D=80) == -2 and att(page=17) == -2
    assert att(width=1 << 28) == -2
    assert att(width=4096, ts=4096) == -3 and b"workspace" in lib.hx_last_error()   # long keys, few rows: split
    assert att(tokens=0, batch=0) == 0
    assert lib.hx_kv4_attention_workspace_bytes(2, 2, 2, 1, 128, 16, 4, 1, 1) == 0
    assert lib.hx_kv4_attention_workspace_bytes(2, 2, 2, 1, 128, 16, 4096, 1, 1) % (2 * 2 * 130 * 4) == 0
    assert lib.hx_kv4_attention_workspace_bytes(0, 2, 2, 1, 128, 16, 4096, 1, 1) == 0


def test_cpu_tensors_are_refused():
    x8, s = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.int8_gemm(x8, x8.t(), s, s)
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.int8_quantize_per_token(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.rms_norm_int8(torch.zeros(2, 4), torch.ones(4))
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.rms_norm_int8(torch.zeros(2, 4), torch.ones(4), residual=torch.zeros(2, 4))
    c = hx.kv4_cache(2, 16, 1, 64, device="cpu")
    k = torch.zeros(1, 1, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.kv4_write(c, k, k, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.kv4_read(c, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        hx.kv4_attention(k, c, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def test_cache_shapes_and_refusals():
    c = hx.kv4_cache(3, 32, 2, 128, device="meta")
    assert [tuple(t.shape) for t in c] == [(3, 2, 32, 64), (3, 2, 32, 4), (3, 2, 8, 16, 4, 4), (3, 2, 8, 4, 4)]
    assert all(t.dtype == torch.uint8 for t in c)
    for bad in ((3, 32, 2, 96), (3, 24, 2, 64), (3, 8, 2, 64), (-1, 16, 2, 64), (3, 16, 0, 64)):
        with pytest.raises(ValueError):
            hx.kv4_cache(*bad, device="cpu")


def test_shapes_on_meta_tensors():
    m = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="meta")
    q, s = hx.rms_norm_int8(m(2, 3, 64), m(64))
    assert q.shape == (2, 3, 64) and q.dtype == torch.int8 and s.shape == (2, 3, 1) and s.dtype == torch.float32
    q, s, h = hx.rms_norm_int8(m(5, 64), m(64), residual=m(5, 64))
    assert h.shape == (5, 64) and h.dtype == torch.bfloat16
    q, s = hx.int8_quantize_per_token(m(7, 9))
    assert q.shape == (7, 9) and s.shape == (7, 1)
    o = hx.int8_gemm(m(5, 64, dt=torch.int8), m(64, 8, dt=torch.int8), m(5, dt=torch.float32), m(8, dt=torch.float32), out_dtype=torch.float16)
    assert o.shape == (5, 8) and o.dtype == torch.float16
    c = hx.kv4_cache(3, 16, 2, 64, device="meta")
    k, v = hx.kv4_read(c, m(5, dt=torch.int64), torch.float16)
    assert k.shape == v.shape == (5, 2, 64) and k.dtype == torch.float16
    a = hx.kv4_attention(m(4, 6, 64), c, m(4, 2, dt=torch.int32), m(4, dt=torch.int32))
    assert a.shape == (4, 6, 64) and a.dtype == torch.bfloat16
    assert hx.kv4_write(c, m(5, 2, 64), m(5, 2, 64), m(5, dt=torch.int64)) is None


def test_signatures():
    sig = inspect.signature(hx.kv4_attention).parameters
    assert list(sig)[:4] == ["q", "cache", "block_table", "seq_lens"]
    assert all(sig[n].kind is inspect.Parameter.KEYWORD_ONLY for n in ("query_start", "max_query_len", "scale", "causal", "out"))
    assert list(inspect.signature(hx.int8_gemm).parameters) == ["x", "y", "scale_a", "scale_b", "bias", "out_dtype"]


def test_restatement_of_the_format():
    x = torch.tensor([0.0, 0.25, 0.26, 0.75, 1.25, 1.26, 1.75, 2.5, 3.5, 5.0, 5.1, 6.0, 7.9, -0.75, -5.0, 4.0] + [0.0] * 16)
    codes, byte = ref.encode(x)
    assert byte.tolist() == [127]                            # floor(log2 7.9) - 2 = 0
    assert codes[:16].tolist() == [0, 0, 1, 2, 2, 3, 4, 4, 6, 6, 7, 7, 7, 10, 14, 6]
    assert ref.decode(codes, byte)[:16].tolist() == [0, 0, 0.5, 1, 1, 1.5, 2, 2, 4, 4, 6, 6, 6, -1, -4, 4]
    for e in (-149, -140, -127, -126, 0, 127):               # the largest at powers of two and just below
        y = torch.zeros(32)
        y[3] = 2.0**e
        assert ref.encode(y)[1].item() == max(e - 2, -126) + 127
    y = torch.zeros(2, 64)
    y[0, 1], y[1, 40] = float("inf"), float("nan")
    assert ref.encode(y)[1].tolist() == [[255, 1], [1, 255]]
    c = torch.arange(3 * 2 * 16 * 64).reshape(3, 2, 16, 64).remainder(16).to(torch.uint8)
    s = torch.arange(3 * 2 * 16 * 2).reshape(3, 2, 16, 2).to(torch.uint8)
    for values in (False, True):
        a, b = ref.from_layout(*ref.to_layout(c, s, values), values)
        assert torch.equal(a, c) and torch.equal(b, s)
    vc, vs = ref.to_layout(c, s, True)
    assert vc.shape == (3, 2, 4, 16, 4, 2) and vs.shape == (3, 2, 4, 2, 4)
    # piece 5 of token 6 of a head: elements 20 .. 23
    assert vc[1, 0, 1, 5, 2].tolist() == [int(c[1, 0, 6, 20] | c[1, 0, 6, 21] << 4), int(c[1, 0, 6, 22] | c[1, 0, 6, 23] << 4)]


def test_a_modules_weight_and_inputs_that_require_grad_leave_no_graph():
    """no result carries a gradient, whichever of the arguments would"""
    m = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="meta")
    weight = torch.nn.Parameter(m(64))
    x = m(5, 64).requires_grad_()
    f32 = lambda n: m(n, dt=torch.float32).requires_grad_()
    a8, b8 = m(5, 64, dt=torch.int8), m(64, 8, dt=torch.int8)
    c = hx.kv4_cache(3, 16, 2, 64, device="meta")
    kv, q, i32 = m(4, 2, 64).requires_grad_(), m(4, 6, 64).requires_grad_(), lambda *s: m(*s, dt=torch.int32)
    results = [*hx.rms_norm_int8(m(5, 64), weight), *hx.rms_norm_int8(x, weight, residual=m(5, 64)), *hx.rms_norm_int8(x, m(64), residual=x),
               *hx.int8_quantize_per_token(x), hx.int8_gemm(a8, b8, f32(5), f32(8), bias=torch.nn.Parameter(m(8))),
               *hx.kv4_read(c, m(5, dt=torch.int64)), hx.kv4_attention(q, c, i32(4, 2), i32(4)), hx.kv4_attention(q, c, i32(4, 2), i32(4), out=m(4, 6, 64))]
    hx.kv4_write(c, kv, kv, m(4, dt=torch.int64))
    assert not any(t.requires_grad for t in (*results, *c))


def test_a_padded_max_query_plans_what_the_tokens_need():
    """max_query sizes the launch, but no sequence has more new tokens than there are: one token over 32768 keys is split as
    ever, and no count is too large"""
    lib = _lib.load()
    need = lambda tokens, mq: lib.hx_kv4_attention_workspace_bytes(tokens, 1, 64, 8, 128, 64, 512, mq, 1)
    assert need(1, 1) > 0
    assert need(1, 4096) == need(1, 2**62) == need(1, 1)
    assert need(4, 4096) == need(4, 4) > 0
    ab = dict(q=A, qt=8192, qh=128, kc=A, ks=A, vc=A, vs=A, table=A, ts=512, lens=A, start=A, out=A, tokens=1, batch=1, heads=64, kv=8, D=128,
              pages=512, page=64, width=512, mq=4096, scale=0.1, causal=1, dt=1, ws=A, wsb=need(1, 1) - 1)
    assert lib.hx_kv4_attention(*ab.values(), None) == -3 and str(need(1, 1)).encode() in lib.hx_last_error()  # the same plan


def test_which_kernel_a_size_runs():
    """(at 256 compute units, which is what the library takes without a GPU)"""
    lib = _lib.load()
    gemm = lambda m, n, k, a=A, b=A: lib.hx_int8_gemm_path(m, n, k, k, 1, k, a, b)
    assert [gemm(*s) for s in ((16, 28672, 8192), (1, 64, 16384), (16, 300, 1040), (512, 4096, 4096), (128, 8192, 8192), (777, 4096, 4096),
                               (777, 4100, 4112), (200, 4096, 16384), (8192, 8192, 8192), (3500, 2560, 4112))] == [1, 9, 17, 2, 10, 3, 19, 11, 4, 20]
    assert [gemm(*s) for s in ((16, 1024, 8192), (1, 1024, 4096), (16, 2048, 2048), (32, 256, 8192))] == [1] * 4  # splitting costs more than it gives
    assert gemm(8192, 8192, 8191) == 4 and gemm(777, 4100, 4112, A + 1) == 19 and gemm(777, 4100, 4112, A + 1, A + 1) == 3  # copies have whole k-tiles
    assert gemm(0, 4, 4) == 0 and gemm(4, 4, 200000) == 0
    att = lambda t, b, h, kv, d, page, width, mq, dt=1: lib.hx_kv4_attention_path(t, b, h, kv, d, page, width, mq, dt)
    assert att(1, 1, 32, 8, 128, 16, 33, 1) == 1 and att(32, 32, 64, 8, 128, 64, 512, 1) == 9 and att(64, 64, 32, 32, 64, 16, 128, 1) == 1
    assert att(2048, 1, 32, 8, 128, 64, 160, 2048) == 3 and att(1000, 24, 32, 8, 128, 32, 125, 200) == 2
    assert att(2048, 1, 32, 8, 128, 64, 160, 2048, 2) == 1 and att(0, 1, 8, 8, 64, 16, 1, 1) == 0
