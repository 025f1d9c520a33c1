"""Bindings of the block-scaled e4m3 path, 8-bit weights and activations: rows in e4m3 (csrc/kernels/rows_e4m3.cu), their products
(csrc/kernels/gemm_e4m3_sm100.cu; prompts: csrc/kernels/gemm_rows_e4m3_sm100.cu) and what stands around those of experts
(csrc/kernels/experts_e4m3.cu).

Nothing here keeps scratch between calls, so calls on several streams and captured graphs do not touch one another; the kernels run on
the device of their rows, on that device's current stream.  A step of a small model is bound by the host, so arguments go over as one
packed struct or as plain numbers."""
from __future__ import annotations

import ctypes as C
import math
import struct
import weakref

import torch

from . import native as N
from .rows import BLOCK, RowsE4M3

MAX_COLS = 32768               # of a row that is quantised: it stays in registers

# csrc/kernels/rows_e4m3.cuh:RowsGemm, field after field: x, x_scale, w, w_scale, out, out_scale, bias, residual, group_tiles, num_group_tiles,
# col_scale, status | x_ld, out_ld | x_rows, ldx, w_rows, ldw, scale_ld, T, N, K, ldo, out_fp32, ldr, act, gated, dual_off, group_w_rows,
# max_tiles, bn, form | res_scale
ROWS_GEMM = struct.Struct("@12P2q18if")
_P, _I, _L = C.c_void_p, C.c_int, C.c_longlong
# csrc/kernels/rows_e4m3.cu:RowsArgs: x, r, gain, codes, scale, h, y | ldx, ldr, ldc, lds, ldh, ldy | rows, K, r_kind | eps
ROWS_ARGS = struct.Struct("@7P6q3if")
_ARGS = {"xft_rows_e4m3": [C.c_char_p, _P],
         "xft_plan_rows": [_P, _P, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _I, _P],
         "xft_sum_rows": [_P, _I, _P, _P, _I, _P, _P, _P, _P, _I, _I, _P],
         "xft_gather_e4m3": [_P, _L, _P, _L, _P, _P, _I, _I, _P, _L, _P, _L, _P],
         "xft_gemm_rows_e4m3": [C.c_char_p, _P]}
_fns = None


def _lib():
    global _fns
    if _fns is None:
        _fns = N.lib()
        for name, args in _ARGS.items():
            f = getattr(_fns, name)
            f.restype, f.argtypes = _I, args
    return _fns


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _foreign(device) -> bool:
    """Whether `device` is another than the current one, which allocations, stream and launches would go to."""
    return device.index != torch._C._cuda_getDevice()


def new_rows(T, K, beside) -> RowsE4M3:
    """Room for rows on the device of `beside`: codes on a pitch of 16 bytes, which the products' copies want."""
    codes = beside.new_empty((T, (K + 15) // 16 * 16), dtype=torch.float8_e4m3fn)
    return RowsE4M3.of(codes if K % 16 == 0 else codes[:, :K], beside.new_empty((-(-K // BLOCK), T), dtype=torch.float32))


def _pitched(codes):
    """Codes whose rows start on 16 bytes (a copy where they do not)."""
    ld, one = codes.stride()
    if one == 1 and ld % 16 == 0 and codes.data_ptr() % 16 == 0:
        return codes
    T, K = codes.shape
    own = codes.new_empty((T, (K + 15) // 16 * 16))                     # (what lies behind a row is never read)
    if one == 1 and ld % 8 == 0 and K % 8 == 0 and codes.data_ptr() % 8 == 0:
        own.view(torch.int64)[:, :K // 8].copy_(codes.view(torch.int64))     # eight bytes at a time
    else:
        own[:, :K].copy_(codes)
    return own[:, :K]


def _pitch(codes) -> int:
    return codes.stride(0) if codes.shape[0] > 1 else (max(codes.stride(0), codes.shape[1]) + 15) // 16 * 16


def _scales(scale):
    return scale if scale.stride(1) == 1 or scale.shape[1] <= 1 else scale.contiguous()


def rows_e4m3(x, gain=None, eps=0.0, residual=None, want_rows=False):
    """(rows, normalised bf16 rows or None, x + residual or None), see ops.quantize_e4m3 and ops.rmsnorm_e4m3."""
    dev = x.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return rows_e4m3(x, gain, eps, residual, want_rows)
    K = x.shape[-1]
    if x.dtype is not torch.bfloat16 or K % 8 or not 0 < K <= MAX_COLS:
        raise N.KernelError(f"rows in e4m3 are made of bf16 rows of up to {MAX_COLS} columns, a multiple of 8 (got {K} in {x.dtype})")
    whole = x.is_contiguous()
    x2, ldx = (x, K) if whole and x.data_ptr() % 16 == 0 else N._rows2d(x)
    T = x2.numel() // K
    q = new_rows(T, K, x2)
    codes, y, h, r, ldr, kind = q.codes, None, None, 0, 0, 0
    if want_rows:
        y = torch.empty_like(x) if whole else x.new_empty(x.shape)           # (the cheaper of torch's ways where it gives whole rows)
    if residual is not None:
        kind = 2 if residual.dtype is torch.float32 else 1
        if kind == 1 and residual.dtype is not torch.bfloat16:
            raise N.KernelError(f"a residual is bf16 or fp32, not {residual.dtype}")
        r2, ldr = (residual, K) if residual.is_contiguous() and residual.data_ptr() % 16 == 0 else N._rows2d(residual)
        r = r2.data_ptr()
        h = torch.empty_like(x) if whole else x.new_empty(x.shape)
    if gain is not None and (gain.dtype is not torch.float32 or not gain.is_contiguous() or gain.data_ptr() % 16):
        gain = gain.float().clone(memory_format=torch.contiguous_format)
    a = ROWS_ARGS.pack(x2.data_ptr(), r, 0 if gain is None else gain.data_ptr(), codes.data_ptr(), q.scale.data_ptr(), 0 if h is None else h.data_ptr(),
                       0 if y is None else y.data_ptr(), ldx, ldr, (K + 15) // 16 * 16, T, K, K, T, K, kind, eps)
    rc = _lib().xft_rows_e4m3(a, _stream())
    if rc:
        N._check(rc, "rows_e4m3")
    N.Workspace.get(dev).launches += 1
    return q, y, h


def rows_of(x) -> RowsE4M3:
    """What a product of 8-bit rows reads of x; a rank's empty share of the columns has no rows to launch for."""
    return rows_e4m3(x)[0] if x.shape[-1] else new_rows(math.prod(x.shape[:-1]), 0, x)


AFTER_COPY = -2                # csrc/kernels/rows_e4m3.cuh:kRowsFormAfterCopy


def _form(W, w) -> int:
    """How a product of `_weight`'s codes w is launched: a copy that is not kept was made by the launch in front of it."""
    return -1 if w is W.w or W.cache.get("w_pitch16") is w else AFTER_COPY


def _weight(W):
    """The codes of W with rows on 16 bytes; the copy that this may take is kept with the weight (inside a capture it is part of the graph, and
    the product behind it says so, see `_form`)."""
    w = W.w
    ld, one = w.stride()
    if ld % 16 or one != 1 or w.data_ptr() % 16:
        kept = W.cache.get("w_pitch16")
        if kept is None:
            kept = _pitched(w)
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(w.device).synchronize()       # other streams may read it from now on
                W.cache["w_pitch16"] = kept
        w = kept
    return w


def _gemm(q, w, w_scale, out, T, n_out, K, gated=False, dual_off=0, bias=None, act=None, residual=None, res_scale=1.0, out_scale=None,
          tiles=None, n_tiles=None, group_rows=0, max_tiles=0, bn=0, col_scale=None, form=-1):
    codes, scale = _pitched(q.codes), _scales(q.scale)
    ws = N.Workspace.get(codes.device)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    a = ROWS_GEMM.pack(codes.data_ptr(), scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), out.data_ptr(), ptr(out_scale), ptr(bias),
                       ptr(residual), ptr(tiles), ptr(n_tiles), ptr(col_scale), ws.status.data_ptr(),
                       scale.stride(0) if scale.shape[0] > 1 else scale.shape[1], 0 if out_scale is None else out_scale.shape[1],
                       codes.shape[0], _pitch(codes), w.shape[0], _pitch(w), w_scale.shape[1], T, n_out, K,
                       out.stride(0) if out_scale is None else _pitch(out), out.dtype is torch.float32,
                       0 if residual is None else residual.stride(0), N._ACT[act], gated, dual_off, group_rows, max_tiles, bn, form, res_scale)
    rc = _lib().xft_gemm_rows_e4m3(a, _stream())
    if rc:
        N._check(rc, "gemm_rows_e4m3")
    ws.launches += 1


def linear_e4m3(q, W, bias=None, act=None, residual=None, res_scale=1.0, out_dtype=torch.bfloat16):
    dev = q.codes.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return linear_e4m3(q, W, bias, act, residual, res_scale, out_dtype)
    T, K = q.codes.shape
    if residual is not None:
        if residual.dtype is not torch.bfloat16:
            raise N.KernelError(f"the residual of a product is bf16, not {residual.dtype}")
        if residual.dim() != 2:
            residual = residual.reshape(-1, residual.shape[-1])
        if residual.stride(1) != 1:
            residual = residual.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if not K:                                            # a rank's empty share of a row-parallel product
        from . import reference as R
        y = R._act(torch.zeros((T, W.out_features), device=dev) + (0 if bias is None else bias), act)
        return (y if residual is None else y + res_scale * residual.float()).to(out_dtype)
    out = q.codes.new_empty((T, W.out_features), dtype=out_dtype)
    if T:
        w = _weight(W)
        _gemm(q, w, W.scale, out, T, W.out_features, K, False, 0, bias, act, residual, res_scale, form=_form(W, w))
    return out


def linear_gated_e4m3(q, W, act="silu", bias=None) -> RowsE4M3:
    dev = q.codes.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return linear_gated_e4m3(q, W, act, bias)
    T, K = q.codes.shape
    I = W.out_features // 2
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if not K:                                            # no columns, as in linear_e4m3
        from . import reference as R
        return R.linear_gated_e4m3(q, W, act, bias)
    out = new_rows(T, I, q.codes)
    if T and I:
        w = _weight(W)
        _gemm(q, w, W.scale, out.codes, T, I, K, True, I, bias, act, out_scale=out.scale, form=_form(W, w))
    return out


def gated_rows(q, W, act, bias=None):
    """act(g) * u as bf16 rows."""
    T, K = q.shape
    I = W.out_features // 2
    out = torch.empty(T, I, dtype=torch.bfloat16, device=q.device)
    if T:
        w = _weight(W)
        _gemm(q, w, W.scale, out, T, I, K, True, I, bias, act, form=_form(W, w))
    return out


def packed_before(experts):
    """The stacks that an earlier call made of these very experts, kept with the first one's weight; None where there are none."""
    for of, pk in experts[0][0].cache.get("e4m3_packs", ()):
        if len(of) == len(experts) and all(a() is g and b() is d for (a, b), (g, d) in zip(of, experts)):
            return pk
    return None


def pack_experts(experts) -> dict:
    """Stacks of these experts, made once: what a captured graph reads stays, also when another list with the same first expert comes, for as long
    as all of its experts do.  (Each list that lives has stacks of its own; who holds the result holds them longer.)"""
    pk = packed_before(experts)
    if pk is None:
        from . import native_moe
        cache, dev = experts[0][0].cache, experts[0][0].w.device
        if torch.cuda.is_current_stream_capturing():
            raise N.KernelError("experts' weights are stacked before a graph is captured (pack_experts_e4m3), not inside it")
        whole = lambda of: all(a() is not None and b() is not None for a, b in of)
        packs = cache.setdefault("e4m3_packs", [])
        gone = [p for of, p in packs if not whole(of)]                      # nobody can ask for these again
        packs[:] = [(of, p) for of, p in packs if whole(of)]
        if any(p is cache.get("moe_pack") for p in gone):
            del cache["moe_pack"]
        old = cache.get("moe_pack")
        step = lambda s, n: s.data_ptr() + n * s.shape[1]
        if old is not None and "gus" in old and old["E"] == len(experts) and all(
                g.w.data_ptr() == step(old["gu"], e * 2 * old["I"]) and d.w.data_ptr() == step(old["dn"], e * old["H"])
                for e, (g, d) in enumerate(experts)):
            pk = old
        else:
            pk = native_moe._pack_fp8(experts)
            if old is not None:
                cache["moe_pack"] = old
        packs.append(([(weakref.ref(g), weakref.ref(d)) for g, d in experts], pk))
        torch.cuda.current_stream(dev).synchronize()                    # other streams may read them from now on
    return pk


def _tile_rows(avg) -> int:
    """Rows of a tile for experts of `avg` rows on average: 16 and 32 rows on the weight stream, 128 and 256 on the kernel of prompts.  A tile
    with fewer rows reads an expert's weights more often, one with more multiplies rows that are not there.  B200, us with 16 / 32 / 128 / 256
    (64 lies between its neighbours everywhere): 64 experts of 1408 x 2048, average 0.8: 56 / 59 / 86 / 116, 6: 108 / 103 / 135 / 196, 19: 148 /
    126 / 156 / 218, 66: 318 / 224 / 185 / 247, 384: 1630 / 1034 / 431 / 486; 8 of 14336 x 4096, 16: 275 / 273 / 274 / 381, 50: 458 / 330 / 283 /
    394, 1024: - / - / 1712 / 1750, 2048: - / - / 3253 / 3183."""
    return 16 if avg <= 4 else 32 if avg <= 32 else 128 if avg < 1536 else 256


def moe_experts_e4m3(q, idx, w, experts, act="silu", expert_offset=0, packed=None, expected_pairs=None, add=None, out_dtype=torch.float32):
    dev = q.codes.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return moe_experts_e4m3(q, idx, w, experts, act, expert_offset, packed, expected_pairs, add, out_dtype)
    pk = packed or pack_experts(experts)
    (T, H), k = q.codes.shape, idx.shape[1]
    E, I = pk["E"], pk["I"]
    out = q.codes.new_empty((T, H), dtype=out_dtype)
    if T == 0:
        return out
    if I == 0:                                           # a rank's empty share of the experts' features
        return out.zero_() if add is None else out.copy_(add)
    ws, lib, st = N.Workspace.get(dev), _lib(), _stream()
    pairs = T * k
    avg = max(1, ((pairs if expected_pairs is None else min(int(expected_pairs), pairs)) + E - 1) // E)
    bn = _tile_rows(avg)
    max_tiles = (pairs + bn - 1) // bn + E
    # one allocation for everything between the rows and the sum (a step of a small model is bound by the host): the plan's tiles, positions,
    # sources, weights and counts, the gathered rows, the middle rows and the pairs' results
    # A pair's result waits for the sum in fp32; prompts whose result is bf16 let it wait in bf16, half the bytes: 4096 tokens on 6 of 64 experts of
    # 1408 x 2048 388 us and 427 with fp32, 512 on 8 of 64 167 and 186, 300 on 2 of 8 of 14336 x 4096 292 and 294; each pair is then off by half a
    # step of bf16 more (against 64 bits 0.0023 of the result, and 0.0017).  The routing weights come in with the fp32 sum.
    prompt = bn >= 128
    half = prompt and out_dtype is torch.bfloat16
    places, size = [], 0
    for n in (16 * max_tiles, 4 * pairs, 4 * pairs, 4 * pairs, 8, pairs * H, 4 * pairs * (H // BLOCK), pairs * I, 4 * pairs * (I // BLOCK),
              (2 if half else 4) * pairs * H):
        places.append(size)
        size += (n + 255) // 256 * 256
    room = q.codes.new_empty(size, dtype=torch.uint8)
    base = room.data_ptr()
    tiles, pos, src, row_w, meta, xc, xs, hc, hs, ys = [base + p for p in places]
    idx32, w32 = (idx if idx.dtype is torch.int32 else idx.int()).contiguous(), w.float().contiguous()
    N._check(lib.xft_plan_rows(idx32.data_ptr(), w32.data_ptr(), T, k, expert_offset, expert_offset + E, bn, pos, src, row_w, tiles, meta, max_tiles, st),
             "plan_rows")
    codes, scale = _pitched(q.codes), _scales(q.scale)
    N._check(lib.xft_gather_e4m3(codes.data_ptr(), _pitch(codes), scale.data_ptr(), scale.stride(0) if scale.shape[0] > 1 else T, src, meta + 4,
                                 pairs, H, xc, H, xs, pairs, st), "gather_e4m3")
    gu, gus, dn, dns, status = pk["gu"], pk["gus"], pk["dn"], pk["dns"], ws.status.data_ptr()
    a = ROWS_GEMM.pack(xc, xs, gu.data_ptr(), gus.data_ptr(), hc, hs, 0, 0, tiles, meta, 0, status, pairs, pairs, pairs, H, gu.shape[0], H,
                       gus.shape[1], pairs, I, H, I, 0, 0, N._ACT[act], 1, I, 2 * I, max_tiles, bn, -1, 1.0)
    N._check(lib.xft_gemm_rows_e4m3(a, st), "experts' gate_up")
    a = ROWS_GEMM.pack(hc, hs, dn.data_ptr(), dns.data_ptr(), ys, 0, 0, 0, tiles, meta, 0 if prompt else row_w, status, pairs, 0, pairs, I,
                       dn.shape[0], I, dns.shape[1], pairs, H, I, H, not half, 0, 0, 0, 0, H, max_tiles, bn, -1, 1.0)
    N._check(lib.xft_gemm_rows_e4m3(a, st), "experts' down")
    if add is not None and (not add.is_contiguous() or add.data_ptr() % 16):
        add = add.clone(memory_format=torch.contiguous_format)
    add32, add16 = (0, 0) if add is None else (add.data_ptr(), 0) if add.dtype is torch.float32 else (0, add.data_ptr())
    o16, o32 = (out.data_ptr(), 0) if out_dtype is torch.bfloat16 else (0, out.data_ptr())
    N._check(lib.xft_sum_rows(ys, not half, pos, w32.data_ptr() if prompt else 0, k, add32, add16, o32, o16, T, H, st), "sum_rows")
    ws.launches += 5
    return out
