"""Bindings of the block-scaled e4m3 path, 8-bit weights and activations: rows in e4m3 (csrc/kernels/rows_e4m3.cu), their products
(csrc/kernels/gemm_e4m3_sm100.cu; prompts: csrc/kernels/gemm_rows_e4m3_sm100.cu) and the experts' form of both.

Nothing here keeps scratch between calls, so calls on several streams and captured graphs do not touch one another; the kernels run on
the device of their rows, on that device's current stream."""
from __future__ import annotations

import ctypes as C

import torch

from . import native as N
from .rows import BLOCK, RowsE4M3

MAX_COLS = 32768               # of a row that is quantised: it stays in registers


class RowsGemm(C.Structure):
    """Mirror of the struct of the same name in csrc/kernels/rows_e4m3.cuh."""
    _fields_ = [("x", C.c_void_p), ("x_scale", C.c_void_p), ("w", C.c_void_p), ("w_scale", C.c_void_p), ("out", C.c_void_p),
                ("out_scale", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p), ("group_tiles", C.c_void_p),
                ("num_group_tiles", C.c_void_p), ("col_scale", C.c_void_p), ("status", C.c_void_p), ("x_ld", C.c_longlong),
                ("out_ld", C.c_longlong), ("x_rows", C.c_int), ("ldx", C.c_int), ("w_rows", C.c_int), ("ldw", C.c_int),
                ("scale_ld", C.c_int), ("T", C.c_int), ("N", C.c_int), ("K", C.c_int), ("ldo", C.c_int), ("out_fp32", C.c_int),
                ("ldr", C.c_int), ("act", C.c_int), ("gated", C.c_int), ("dual_off", C.c_int), ("group_w_rows", C.c_int),
                ("max_tiles", C.c_int), ("bn", C.c_int), ("form", C.c_int), ("res_scale", C.c_float)]


_ready = False


def _lib():
    global _ready
    lib = N.lib()
    if not _ready:
        for fn in ("xft_rows_e4m3", "xft_gather_e4m3", "xft_gemm_rows_e4m3", "xft_moe_plan", "xft_moe_combine", "xft_moe_combine_bf16"):
            getattr(lib, fn).restype = C.c_int
        _ready = True
    return lib


def _on(device):
    """The device of the rows as the current one, for launches, allocations and the stream."""
    return torch.cuda.device(device)


def _foreign(t) -> bool:
    return t.device.index != torch._C._cuda_getDevice()


def _ptr(t):
    return None if t is None else t.data_ptr()


def new_rows(T, K, device) -> RowsE4M3:
    """Room for rows: codes on a pitch of 16 bytes, which the products' copies want."""
    codes = torch.empty(T, (K + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=device)
    return RowsE4M3(codes if K % 16 == 0 else codes[:, :K], torch.empty(-(-K // BLOCK), T, dtype=torch.float32, device=device))


def _pitched(codes):
    """Codes whose rows start on 16 bytes (a copy where they do not)."""
    if codes.stride(1) == 1 and codes.stride(0) % 16 == 0 and codes.data_ptr() % 16 == 0:
        return codes
    T, K = codes.shape
    own = torch.zeros(T, (K + 15) // 16 * 16, dtype=torch.uint8, device=codes.device)
    own[:, :K] = codes.view(torch.uint8)
    return own.view(torch.float8_e4m3fn)[:, :K]


def _pitch(codes) -> int:
    return codes.stride(0) if codes.shape[0] > 1 else (max(codes.stride(0), codes.shape[1]) + 15) // 16 * 16


def _scales(scale):
    return scale if scale.stride(1) == 1 or scale.shape[1] <= 1 else scale.contiguous()


def rows_e4m3(x, gain=None, eps=0.0, residual=None, want_rows=False):
    """(rows, normalised bf16 rows or None, x + residual or None), see ops.quantize_e4m3 and ops.rmsnorm_e4m3."""
    if _foreign(x):
        with _on(x.device):
            return rows_e4m3(x, gain, eps, residual, want_rows)
    x2, ldx = N._rows2d(x)
    T, K = x2.shape
    if x2.dtype != torch.bfloat16 or K % 8 or not 0 < K <= MAX_COLS:
        raise N.KernelError(f"rows in e4m3 are made of bf16 rows of up to {MAX_COLS} columns, a multiple of 8 (got {K} in {x2.dtype})")
    q = new_rows(T, K, x.device)
    y = torch.empty(T, K, dtype=torch.bfloat16, device=x.device) if want_rows else None
    h, r2, ldr, kind = None, None, 0, 0
    if residual is not None:
        if residual.dtype not in (torch.bfloat16, torch.float32):
            raise N.KernelError(f"a residual is bf16 or fp32, not {residual.dtype}")
        r2, ldr = N._rows2d(residual)
        kind = 2 if r2.dtype == torch.float32 else 1
        h = torch.empty(T, K, dtype=torch.bfloat16, device=x.device)
    if gain is not None and (gain.dtype != torch.float32 or not gain.is_contiguous() or gain.data_ptr() % 16):
        gain = gain.float().clone(memory_format=torch.contiguous_format)
    L = C.c_longlong
    N._check(_lib().xft_rows_e4m3(N._p(x2), L(ldx), N._p(r2), L(ldr), kind, N._p(gain), C.c_float(eps), T, K, N._p(q.codes), L(_pitch(q.codes)),
                                  N._p(q.scale), L(T), N._p(h), L(K), N._p(y), L(K), N._stream()), "rows_e4m3")
    N.Workspace.get(x.device).launches += 1
    shape = x.shape
    return q, y if y is None else y.view(shape), h if h is None else h.view(shape)


def _weight(W):
    """The codes of W with rows on 16 bytes; the copy that this may take is kept with the weight."""
    w = W.w
    if w.stride(0) % 16 or w.data_ptr() % 16 or w.stride(1) != 1:
        kept = W.cache.get("w_pitch16")
        if kept is None:
            kept = W.cache["w_pitch16"] = _pitched(w)
        w = kept
    return w


def _gemm(q, w, w_scale, out, T, n_out, K, gated=False, dual_off=0, bias=None, act=None, residual=None, res_scale=1.0, out_scale=None,
          tiles=None, n_tiles=None, group_rows=0, max_tiles=0, bn=0, col_scale=None, form=-1):
    codes, scale = _pitched(q.codes), _scales(q.scale)
    ws = N.Workspace.get(codes.device)
    a = RowsGemm()
    a.x, a.x_scale, a.w, a.w_scale = codes.data_ptr(), scale.data_ptr(), w.data_ptr(), w_scale.data_ptr()
    a.out, a.out_scale, a.bias, a.residual = out.data_ptr(), _ptr(out_scale), _ptr(bias), _ptr(residual)
    a.group_tiles, a.num_group_tiles, a.col_scale, a.status = _ptr(tiles), _ptr(n_tiles), _ptr(col_scale), ws.status.data_ptr()
    a.x_ld = scale.stride(0) if scale.shape[0] > 1 else scale.shape[1]
    a.out_ld = 0 if out_scale is None else out_scale.shape[1]
    a.x_rows, a.ldx, a.w_rows, a.ldw, a.scale_ld = codes.shape[0], _pitch(codes), w.shape[0], _pitch(w), w_scale.shape[1]
    a.T, a.N, a.K, a.ldo, a.out_fp32 = T, n_out, K, _pitch(out) if out_scale is not None else out.stride(0), int(out.dtype == torch.float32)
    a.ldr, a.act = 0 if residual is None else residual.stride(0), N._ACT[act]
    a.gated, a.dual_off, a.group_w_rows, a.max_tiles, a.bn, a.form, a.res_scale = int(gated), dual_off, group_rows, max_tiles, bn, form, res_scale
    N._check(_lib().xft_gemm_rows_e4m3(C.byref(a), N._stream()), "gemm_rows_e4m3")
    ws.launches += 1


def linear_e4m3(q, W, bias=None, act=None, residual=None, res_scale=1.0, out_dtype=torch.bfloat16):
    if _foreign(q):
        with _on(q.device):
            return linear_e4m3(q, W, bias, act, residual, res_scale, out_dtype)
    T, K = q.shape
    if residual is not None:
        residual = residual.reshape(-1, residual.shape[-1])
        if residual.dtype != torch.bfloat16:
            raise N.KernelError(f"the residual of a product is bf16, not {residual.dtype}")
        if residual.stride(1) != 1:
            residual = residual.contiguous()
    out = torch.empty(T, W.out_features, dtype=out_dtype, device=q.device)
    if T:
        _gemm(q, _weight(W), W.scale, out, T, W.out_features, K, False, 0, bias, act, residual, res_scale)
    return out


def linear_gated_e4m3(q, W, act="silu", bias=None) -> RowsE4M3:
    if _foreign(q):
        with _on(q.device):
            return linear_gated_e4m3(q, W, act, bias)
    T, K = q.shape
    I = W.out_features // 2
    out = new_rows(T, I, q.device)
    if T:
        _gemm(q, _weight(W), W.scale, out.codes, T, I, K, True, I, bias, act, out_scale=out.scale)
    return out


def gated_rows(q, W, act, bias=None):
    """act(g) * u as bf16 rows."""
    T, K = q.shape
    I = W.out_features // 2
    out = torch.empty(T, I, dtype=torch.bfloat16, device=q.device)
    if T:
        _gemm(q, _weight(W), W.scale, out, T, I, K, True, I, bias, act)
    return out


def pack_experts(experts) -> dict:
    from . import native_moe
    return native_moe.pack_experts(experts)


def moe_experts_e4m3(q, idx, w, experts, act="silu", expert_offset=0, packed=None, expected_pairs=None, add=None, out_dtype=torch.float32):
    if _foreign(q):
        with _on(q.device):
            return moe_experts_e4m3(q, idx, w, experts, act, expert_offset, packed, expected_pairs, add, out_dtype)
    pk = packed or pack_experts(experts)
    (T, H), k, dev = q.shape, idx.shape[1], q.device
    E, I = pk["E"], pk["I"]
    out = torch.empty(T, H, dtype=out_dtype, device=dev)
    if T == 0:
        return out
    ws, lib = N.Workspace.get(dev), _lib()
    pairs = T * k
    avg = max(1, ((pairs if expected_pairs is None else min(int(expected_pairs), pairs)) + E - 1) // E)
    bn = 16 if avg <= 16 else 32 if avg <= 32 else 64 if avg <= 64 else 128 if avg < 512 else 256
    max_tiles = (pairs + bn - 1) // bn + E
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)
    pos, src, tiles, meta = i32(pairs), i32(pairs), i32(max_tiles, 4), i32(2)
    row_w = torch.empty(pairs, dtype=torch.float32, device=dev)
    idx32, w32 = (idx if idx.dtype == torch.int32 else idx.int()).contiguous(), w.float().contiguous()
    N._check(lib.xft_moe_plan(N._p(idx32), N._p(w32), T, k, expert_offset, expert_offset + E, bn, N._p(pos), N._p(src), N._p(row_w),
                              N._p(tiles), N._p(meta), max_tiles, pairs, N._stream()), "moe_plan")
    codes, scale, L = _pitched(q.codes), _scales(q.scale), C.c_longlong
    xs, h1 = new_rows(pairs, H, dev), new_rows(pairs, I, dev)
    N._check(lib.xft_gather_e4m3(N._p(codes), L(_pitch(codes)), N._p(scale), L(scale.stride(0) if scale.shape[0] > 1 else T), N._p(src),
                                 N._p(meta[1:]), pairs, H, N._p(xs.codes), L(_pitch(xs.codes)), N._p(xs.scale), L(pairs), N._stream()), "gather_e4m3")
    group = dict(tiles=tiles, n_tiles=meta, max_tiles=max_tiles, bn=bn)
    _gemm(xs, pk["gu"], pk["gus"], h1.codes, pairs, I, H, True, I, act=act, out_scale=h1.scale, group_rows=2 * I, **group)
    add32, add16 = (None, None) if add is None else (add.contiguous(), None) if add.dtype == torch.float32 else (None, add.contiguous())
    o16, o32 = (out, None) if out_dtype == torch.bfloat16 else (None, out)
    if bn >= 128:
        # prompts: a pair's row waits for the sum in bf16, half the bytes; the routing weights come in with the fp32 sum
        ys = torch.empty(pairs, H, dtype=torch.bfloat16, device=dev)
        _gemm(h1, pk["dn"], pk["dns"], ys, pairs, H, I, group_rows=H, **group)
        N._check(lib.xft_moe_combine_bf16(N._p(ys), N._p(pos), N._p(w32), k, N._p(add32), N._p(add16), H, N._p(o16), N._p(o32), T, H, N._stream()),
                 "moe_combine")
    else:
        ys = torch.empty(pairs, H, dtype=torch.float32, device=dev)
        _gemm(h1, pk["dn"], pk["dns"], ys, pairs, H, I, group_rows=H, col_scale=row_w, **group)
        N._check(lib.xft_moe_combine(N._p(ys), N._p(pos), k, N._p(add32), N._p(add16), H, N._p(o16), N._p(o32), T, H, N._stream()), "moe_combine")
    ws.launches += 3
    return out
