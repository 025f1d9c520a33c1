"""Op entry points.  Device switch only: CPU tensors run `ops.reference` (pure PyTorch),
CUDA tensors run the hand-written sm_100a kernels of `ops.native` (libxft_b200_kernels.so).

There is no silent fallback on a GPU: if the kernel library is missing or an op has no
kernel for the requested variant, the call raises.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import reference as R
from .rows import BLOCK as _BLOCK, RowsE4M3

_native = None


def _nat():
    global _native
    if _native is None:
        import importlib
        _native = importlib.import_module(__name__ + ".native")
    return _native


def _nat_latent():
    from . import native_latent
    return native_latent


def _cuda(t: torch.Tensor) -> bool:
    return t.is_cuda


# -- embedding / norms ----------------------------------------------------------------------
def embedding(ids, table, scale=1.0, out_dtype=torch.float32, pos_table=None, positions=None, pos_offset=0):
    if _cuda(table):
        return _nat().embedding(ids, table, scale, out_dtype, pos_table, positions, pos_offset)
    return R.embedding(ids, table, scale, out_dtype, pos_table, positions, pos_offset)


def rmsnorm(x, w, eps, residual=None):
    if _cuda(x):
        return _nat().rmsnorm(x, w, eps, residual)
    return R.rmsnorm(x, w, eps, residual)


def layernorm(x, w, b, eps):
    if _cuda(x):
        return _nat().layernorm(x, w, b, eps)
    return R.layernorm(x, w, b, eps)


def residual_norm(x, y, post, nxt, eps, kind="layer", rows=None, h_dtype=torch.bfloat16, ids=None, table=None, keep_x=True,
                  embed_scale=1.0, mult=1.0, add=None, raw=False, carry=1.0, post_sum=False):
    """One step of a 32-bit residual stream in one launch: x (or table[ids] * embed_scale) = carry * x + mult * norm(y) with
    `post` = (gain, bias or None) (plain y without it) + the vector `add`, then h = norm(x) with `nxt` for the next product
    (`raw`: x itself).  `post_sum`: `post` normalises the sum instead of y, and its output is the stream.  Returns (x, h); on a GPU x is updated in place unless `rows` selects rows, and buffers are as wide as x (a
    multiple of 8, padding zero)."""
    impl = _nat().residual_norm if _cuda(x if x is not None else table) else R.residual_norm
    return impl(x, y, post, nxt, eps, kind, rows, h_dtype, ids, table, keep_x, embed_scale, mult, add, raw, carry, post_sum)


# -- GEMMs ---------------------------------------------------------------------------------
_Env = None


def _verbose() -> bool:
    global _Env
    if _Env is None:
        from ..utils.flags import Env as _Env
    return _Env.get().verbose >= 1


def _timed(kernel: str, x, W, fn):
    """XFT_VERBOSE >= 1: run one GEMM-shaped op between two time stamps (device-synchronised on a GPU) and print the
    reference's per-call line ``xft_verbose,exec,<dev>,api,<kernel>,m<M>n<N>k<K>,<ms>`` (src/utils/verbose.h:24-83).
    The decode graph runner steps aside while this is on, so every call is a real launch."""
    import math
    import time
    from ..utils import log
    cuda = _cuda(x)
    if cuda:
        torch.cuda.synchronize(x.device)
    t0 = time.perf_counter()
    y = fn()
    if cuda:
        torch.cuda.synchronize(x.device)
    ms = (time.perf_counter() - t0) * 1e3
    log.verbose_line("gpu" if cuda else "cpu", kernel, math.prod(x.shape[:-1]), W.out_features, x.shape[-1], ms)
    return y


def linear(x, W, bias=None, act=None, residual=None, res_scale=1.0, out_dtype=None, times=None, out=None):
    """act(x W^T + bias) + res_scale * residual, or with `times` [T, out] act(x W^T + bias) * times.  x may be rows in e4m3 where W is
    (see linear_e4m3).  `out`: rows to write into.  act "softcap": res_scale * tanh(. / res_scale)."""
    if isinstance(x, RowsE4M3):
        if out is not None or times is not None:
            raise ValueError("linear: products of rows in e4m3 have no `out` and no `times`")
        return linear_e4m3(x, W, bias, act, residual, res_scale, out_dtype)
    if out is not None:
        assert residual is None and times is None
        return (_nat() if _cuda(x) else R).linear_into(x, W, bias, act, out)
    if times is not None:
        return (_nat() if _cuda(x) else R).linear_times(x, W, bias, act, times)
    if _verbose():
        name = "gemm" + ("_bias" if bias is not None else "") + (f"_{act}" if act else "") + \
            ("_residual" if residual is not None else "")
        impl = _nat().linear if _cuda(x) else R.linear
        return _timed(name, x, W, lambda: impl(x, W, bias, act, residual, res_scale, out_dtype))
    if _cuda(x):
        return _nat().linear(x, W, bias, act, residual, res_scale, out_dtype)
    return R.linear(x, W, bias, act, residual, res_scale, out_dtype)


def _linear_rms(x, W, eps, bias, act, gated, out_dtype):
    if _cuda(x):
        return _nat().linear_rms(x, W, eps, bias, act, gated, out_dtype)
    h = R.rmsnorm(x, torch.ones(x.shape[-1], dtype=torch.float32), eps)
    return R.linear_gated(h, W, act, bias) if gated else R.linear(h, W, bias, act, None, 1.0, out_dtype)


def linear_rms(x, W, eps, bias=None, act=None, gated=False, out_dtype=None):
    """RMSNorm(x) @ W^T for a weight whose columns already carry the norm's gain (loader.fold_norm_gain)."""
    if _verbose():
        return _timed("rmsnorm_gemm" + ("_gated" if gated else ""), x, W,
                      lambda: _linear_rms(x, W, eps, bias, act, gated, out_dtype))
    return _linear_rms(x, W, eps, bias, act, gated, out_dtype)


def norm_linear(x, gain, eps, W, bias=None, act=None, gated=False):
    """RMSNorm(x; gain) @ W^T: as rmsnorm and linear (or linear_gated) after each other, in fewer launches where the rows are quantised.
    Weights of kind "fp8a" give the gated form in e4m3 (RowsE4M3) where its halves have a multiple of 128 rows."""
    if W.kind == "fp8a":
        q = rmsnorm_e4m3(x, gain, eps)[0]
        if gated and W.out_features % (2 * _BLOCK) == 0:
            return linear_gated_e4m3(q, W, act, bias)
        y = linear_e4m3(q, W, bias, None if gated else act)
        return gated_act(y, act) if gated else y
    if _verbose() or not _cuda(x):
        h = rmsnorm(x, gain, eps)
        return linear_gated(h, W, act, bias) if gated else linear(h, W, bias, act)
    return _nat().norm_linear(x, gain, eps, W, bias, act, gated)


def linear_gated(x, W, act="silu", bias=None, limit=0.0):
    """act(g) * u with (g | u) = x W^T + bias; act "clamped": g = min(g, limit), u = u clamped to +-limit, and the result is
    g sigmoid(1.702 g) (u + 1)."""
    impl = _nat().linear_gated if _cuda(x) else R.linear_gated
    if _verbose():
        return _timed(f"gemm_gated_{act}", x, W, lambda: impl(x, W, act, bias, limit))
    return impl(x, W, act, bias, limit)


# -- 8-bit weights and activations ------------------------------------------------------------
_ROW_ACTS = (None, "none", "relu", "silu", "gelu", "gelu_tanh", "gelu_new", "gelu_pytorch_tanh", "relu2", "gelu_erf", "tanh", "swiglu")


_e4m3 = None


def _native_e4m3():
    global _e4m3
    if _e4m3 is None:
        from . import native_e4m3 as _e4m3
    return _e4m3


def _same_device(what, first, *tensors):
    d = first.device
    for t in tensors:
        if t is not None and t.device != d:
            raise ValueError(f"{what}: tensors on {d} and on {t.device}")


def _check_rows_e4m3(what, q, W, act):
    if not isinstance(q, RowsE4M3):
        raise ValueError(f"{what} multiplies rows in e4m3 (RowsE4M3), not {type(q).__name__}")
    _check_e4m3_weight(what, W)
    if q.codes.shape[1] != W.in_features:
        raise ValueError(f"{what}: rows of {q.shape[1]} columns and weights of {W.in_features}")
    if act not in _ROW_ACTS:
        raise ValueError(f"{what}: no activation {act!r}")


def _check_e4m3_weight(what, W):
    if W.kind not in ("fp8", "fp8a") or W.block != _BLOCK:
        raise ValueError(f"{what}: weights are e4m3 with a scale for each block of {_BLOCK}, not {W.kind}")
    n, k, s = W.out_features, W.in_features, W.scale
    if s.shape != (-(-n // _BLOCK), -(-k // _BLOCK)) or s.dtype is not torch.float32 or not s.is_contiguous() or W.w.shape != (n, k) \
            or W.w.dtype is not torch.float8_e4m3fn:
        raise ValueError(f"{what}: weights {tuple(W.w.shape)} in {W.w.dtype} with block scales {tuple(s.shape)} in {s.dtype} (contiguous: "
                         f"{s.is_contiguous()}) for [{n}, {k}] in e4m3")


def quantize_e4m3(x) -> RowsE4M3:
    """Rows x [.., K] in e4m3 with a scale for each 128 columns (`RowsE4M3`, [T, K]): codes e4m3(x * (448 / a)), scales a / 448, a = max
    |x| of the block, at least 2^-100.  A value that is not finite becomes the code of NaN."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_e4m3: rows of {tuple(x.shape)}")
    if _cuda(x):
        return _native_e4m3().rows_e4m3(x)[0]
    return R.quantize_e4m3(x.reshape(-1, x.shape[-1]))


def rmsnorm_e4m3(x, w, eps, residual=None, want_rows=False):
    """RMSNorm(x + residual) * w on its way into products of 8-bit rows, in one launch: (rows in e4m3, the normalised rows in x's type or
    None, x + residual or None).  The sum is rounded once, to x's type, and the norm is of what was rounded; codes are taken from the
    fp32 norm.  `residual`: bf16 or fp32 (CPU: any float type), the shape of x.  `want_rows`: for what reads the norm beside the products."""
    if x.dim() < 1 or w.shape != x.shape[-1:]:
        raise ValueError(f"rmsnorm_e4m3: gain {tuple(w.shape)} of rows {tuple(x.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"rmsnorm_e4m3: residual {tuple(residual.shape)} of rows {tuple(x.shape)}")
    _same_device("rmsnorm_e4m3", x, w, residual)
    if _cuda(x):
        return _native_e4m3().rows_e4m3(x, w, eps, residual, want_rows)
    return R.rmsnorm_e4m3(x, w, eps, residual, want_rows)


def linear_e4m3(q, W, bias=None, act=None, residual=None, res_scale=1.0, out_dtype=None):
    """act(rows W^T + bias) + res_scale * residual of rows in e4m3 and e4m3 weights (kinds "fp8" and "fp8a"): sums of 128 columns are
    scaled and added in fp32.  `out_dtype`: bf16 or fp32; the activation type of the device by default (bf16 on a GPU)."""
    _check_rows_e4m3("linear_e4m3", q, W, act)
    T, N = q.codes.shape[0], W.out_features
    if bias is not None and (bias.shape != (N,) or bias.dtype is not torch.float32):
        raise ValueError(f"linear_e4m3: the bias of {N} features is fp32 [{N}], not {tuple(bias.shape)} in {bias.dtype}")
    if residual is not None and (residual.shape[-1] != N or residual.numel() != T * N):
        raise ValueError(f"linear_e4m3: residual {tuple(residual.shape)} of a result [{T}, {N}]")
    if out_dtype not in (None, torch.bfloat16, torch.float32):
        raise ValueError(f"linear_e4m3: results are bf16 or fp32, not {out_dtype}")
    _same_device("linear_e4m3", q.codes, W.w, W.scale, bias, residual)
    if not q.codes.is_cuda:
        return R.linear_e4m3(q, W, bias, act, residual, res_scale, out_dtype or torch.float32)
    if _verbose():
        return _timed("gemm_e4m3", q, W, lambda: _native_e4m3().linear_e4m3(q, W, bias, act, residual, res_scale, out_dtype or torch.bfloat16))
    return _native_e4m3().linear_e4m3(q, W, bias, act, residual, res_scale, out_dtype or torch.bfloat16)


def linear_gated_e4m3(q, W, act="silu", bias=None) -> RowsE4M3:
    """act(g) * u with (g | u) = rows W^T + bias, as rows in e4m3 for the next product: quantised from fp32, a scale for each 128
    features.  The two halves of W have a multiple of 128 rows each."""
    _check_rows_e4m3("linear_gated_e4m3", q, W, act)
    if W.out_features % (2 * _BLOCK):
        raise ValueError(f"linear_gated_e4m3: gate and up have a multiple of {_BLOCK} features each, not {W.out_features / 2:g}")
    if bias is not None and (bias.shape != (W.out_features,) or bias.dtype is not torch.float32):
        raise ValueError(f"linear_gated_e4m3: the bias is fp32 [{W.out_features}], not {tuple(bias.shape)} in {bias.dtype}")
    _same_device("linear_gated_e4m3", q.codes, W.w, W.scale, bias)
    impl = _native_e4m3().linear_gated_e4m3 if q.is_cuda else R.linear_gated_e4m3
    return _timed(f"gemm_e4m3_gated_{act}", q, W, lambda: impl(q, W, act, bias)) if _verbose() else impl(q, W, act, bias)


def pack_experts_e4m3(experts):
    """The stacked weights of a list of experts, (gate | up, down) each, that `moe_experts_e4m3` takes as `packed`; made once, the experts'
    own weights become views of the stacks.  They are kept with the first expert for as long as all experts of the list live; a graph that was
    captured over them needs those, or this result, for as long.  None on a CPU."""
    if not experts:
        raise ValueError("pack_experts_e4m3: no experts")
    for g, d in experts:
        _check_e4m3_weight("pack_experts_e4m3", g)
        _check_e4m3_weight("pack_experts_e4m3", d)
        _same_device("pack_experts_e4m3", experts[0][0].w, g.w, g.scale, d.w, d.scale)
        if d.in_features % _BLOCK or d.out_features % _BLOCK or (g.in_features, g.out_features) != (d.out_features, 2 * d.in_features):
            raise ValueError(f"pack_experts_e4m3: experts of widths that are multiples of {_BLOCK}, gate and up [2 I, H], down [H, I]; not "
                             f"[{g.out_features}, {g.in_features}] and [{d.out_features}, {d.in_features}]")
        if (d.in_features, d.out_features) != (experts[0][1].in_features, experts[0][1].out_features):
            raise ValueError("pack_experts_e4m3: experts of different sizes")
    return _native_e4m3().pack_experts(experts) if experts[0][0].w.is_cuda else None


def moe_experts_e4m3(q, idx, w, experts, act="silu", expert_offset=0, packed=None, expected_pairs=None, add=None, out_dtype=torch.float32):
    """sum_k w[t, k] down_e(act(gate_e q_t) * up_e q_t) (+ `add`, fp32 or bf16) over the local experts e = idx[t, k] - expert_offset of
    rows in e4m3, the middle rows in e4m3 too; experts outside the list (or -1) add nothing.  `out_dtype`: fp32, with sums and the experts'
    parts of them in fp32, or bf16, where a GPU rounds a part to bf16 before it is weighted and added if an expert has more than 32 rows on
    average.  That average comes from `expected_pairs` where that is given.  Other arguments as in `moe_experts`."""
    if not isinstance(q, RowsE4M3):
        raise ValueError(f"moe_experts_e4m3 multiplies rows in e4m3 (RowsE4M3), not {type(q).__name__}")
    T, H = q.shape
    if idx.dim() != 2 or idx.shape[0] != T or idx.shape[1] < 1 or idx.shape != w.shape:
        raise ValueError(f"moe_experts_e4m3: experts {tuple(idx.shape)} and weights {tuple(w.shape)} of {T} rows")
    if add is not None and (tuple(add.shape) != (T, H) or add.dtype not in (torch.float32, torch.bfloat16)):
        raise ValueError(f"moe_experts_e4m3: what is added is [{T}, {H}] in fp32 or bf16, not {tuple(add.shape)} in {add.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"moe_experts_e4m3: results are bf16 or fp32, not {out_dtype}")
    if act not in _ROW_ACTS:
        raise ValueError(f"moe_experts_e4m3: no activation {act!r}")
    if not experts:
        raise ValueError("moe_experts_e4m3: no experts")
    cuda = q.is_cuda
    if packed is None:                                   # packed before: the experts were looked at then
        packed = cuda and _native_e4m3().packed_before(experts) or pack_experts_e4m3(experts)
    elif "gus" not in packed or packed["E"] != len(experts):
        raise ValueError("moe_experts_e4m3: `packed` is not of these e4m3 experts (pack_experts_e4m3)")
    if experts[0][1].out_features != H:
        raise ValueError(f"moe_experts_e4m3: rows of {H} columns and experts of {experts[0][1].out_features}")
    _same_device("moe_experts_e4m3", q.codes, idx, w, add, experts[0][0].w)
    if not cuda:
        return R.moe_experts_e4m3(q, idx, w, experts, act, expert_offset, add, out_dtype)
    return _native_e4m3().moe_experts_e4m3(q, idx, w, experts, act, expert_offset, packed, expected_pairs, add, out_dtype)


def linear_parts(x, W, n, out):
    """`n` products side by side: part i of x's columns with rows i of W's n equal parts, into part i of `out`'s columns."""
    impl = _native_linear().linear_parts if _cuda(x) else R.linear_parts
    return impl(x, W, n, out)


def gated_act(gu, act="silu"):
    if _cuda(gu):
        return _nat().gated_act(gu, act)
    return R.gated_act(gu, act)


# -- attention -----------------------------------------------------------------------------
def qkv_rope_cache(qkv, hq, hkv, d, positions, table, rot_dim, style, kc, vc, ks, vs, slots,
                   q_scale=None, q_norm_w=None, k_norm_w=None, eps=1e-6, rot_offset=0, dv=None):
    """Split packed qkv [T,(hq+2hkv)*d] (value heads of size `dv` when given; hkv = 0: query heads only), optional per-head q/k RMSNorm (Qwen3), RoPE on q and k,
    append k/v to the paged cache at `slots` (int8-quantising when scales are given); returns
    q [T,hq,d].  One kernel on the GPU (reference: QKPO + storeKVCache,
    src/layers/attention.h:560-640, src/kernels/attention_kernels.h:45-69)."""
    if _cuda(qkv):
        return _nat().qkv_rope_cache(qkv, hq, hkv, d, positions, table, rot_dim, style, kc, vc, ks, vs, slots,
                                       q_scale, q_norm_w, k_norm_w, eps, rot_offset, dv)
    T = qkv.shape[0]
    q = qkv[:, : hq * d].reshape(T, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].reshape(T, hkv, d)
    v = qkv[:, (hq + hkv) * d:].reshape(T, hkv, dv or d)
    if q_norm_w is not None:
        q = R.rmsnorm(q, q_norm_w, eps)
        k = R.rmsnorm(k, k_norm_w, eps)
    if table is not None and rot_dim > 0:
        q, k = R.rope_apply(q, k, positions, table, rot_dim, style, rot_offset, q_scale)
    elif q_scale is not None:
        q = (q.float() * q_scale[:, None, None]).to(q.dtype)
    if hkv > 0:
        R.kv_cache_write(k, v, kc, vc, slots, ks, vs)
    return q.contiguous()


def qkv_rope2d_cache(qkv, hq, hkv, d, positions, positions2, table, kc, vc, ks, vs, slots):
    """ChatGLM-1's two-stream rotary with the cache append: the first half of every q / k head turns by `positions`,
    the second half by `positions2` (block positions), both from one table [max_pos, d/2]; k / v go to the paged cache
    at `slots`; returns q [T,hq,d].  One kernel on the GPU (reference: src/layers/rope_2d.cpp,
    src/models/chatglm.cpp:118-206)."""
    if _cuda(qkv):
        return _nat().qkv_rope2d_cache(qkv, hq, hkv, d, positions, positions2, table, kc, vc, ks, vs, slots)
    T = qkv.shape[0]
    q = qkv[:, : hq * d].reshape(T, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].reshape(T, hkv, d)
    v = qkv[:, (hq + hkv) * d:].reshape(T, hkv, d)
    half = d // 2
    q, k = R.rope_apply(q, k, positions, table, half, "half", 0)
    q, k = R.rope_apply(q, k, positions2, table, half, "half", half)
    R.kv_cache_write(k, v, kc, vc, slots, ks, vs)
    return q.contiguous()


def can_fuse_qkv_rope(W, T, D, kc, ks, q_norm_w, k_norm_w, style) -> bool:
    """True when the QKV product, RoPE and the cache append can run as one step (GPU, decode sizes)."""
    return _cuda(kc) and _nat().can_fuse_qkv_rope(W, T, D, kc, ks, q_norm_w, k_norm_w, style)


def qkv_linear_rope_cache(x, W, bias, rms_eps, hq, hkv, positions, table, rot_dim, style, kc, vc, slots, q_scale=None):
    """QKV product with split + RoPE + paged cache append as its epilogue; returns q [T, hq, D].  GPU only: callers
    ask can_fuse_qkv_rope first and otherwise run linear / linear_rms followed by qkv_rope_cache."""
    return _nat().qkv_linear_rope_cache(x, W, bias, rms_eps, hq, hkv, positions, table, rot_dim, style, kc, vc, slots,
                                        q_scale)


def paged_attention(q, kc, vc, block_table, cu_q, kv_lens, scale, ks=None, vs=None, slopes=None,
                    causal=True, prefix_lm_lens=None, group=None, q_off=0, meta=None, softcap=0.0, window=0, keep_first=0,
                    sinks=None):
    """Attention of a ragged batch over the paged cache; `softcap`, `window` with `keep_first`, and `sinks` as in
    `reference.paged_attention`."""
    if _cuda(q):
        return _nat().paged_attention(q, kc, vc, block_table, cu_q, kv_lens, scale, ks, vs, slopes,
                                        causal, prefix_lm_lens, group, q_off, meta, softcap, window, keep_first, sinks)
    return R.paged_attention(q, kc, vc, block_table, cu_q, kv_lens, scale, ks, vs, slopes, causal,
                             prefix_lm_lens, group, q_off, softcap, window, keep_first, sinks)


def mla_attention(q_nope, q_rope, latent_cache, block_table, cu_q, kv_lens, w_uk, w_uv, scale, absorbed=True,
                  meta=None):
    if _cuda(q_nope):
        return _nat().mla_attention(q_nope, q_rope, latent_cache, block_table, cu_q, kv_lens, w_uk, w_uv,
                                      scale, absorbed, meta)
    return R.mla_attention(q_nope, q_rope, latent_cache, block_table, cu_q, kv_lens, w_uk, w_uv, scale, absorbed)


def rope_apply(q, k, positions, table, rot_dim, style="half", rot_offset=0, q_scale=None):
    if _cuda(q):
        return _nat().rope_apply(q, k, positions, table, rot_dim, style, rot_offset, q_scale)
    return R.rope_apply(q, k, positions, table, rot_dim, style, rot_offset, q_scale)


def latent_cache_write(latent, cache, slots):
    """latent [T, kv_lora+rope] -> cache [nb,1,block,kv_lora+rope] at `slots`."""
    if _cuda(latent):
        return _nat().latent_cache_write(latent, cache, slots)
    blk = cache.shape[2]
    cache[(slots // blk).long(), 0, (slots % blk).long()] = latent.to(cache.dtype)


def mla_prep(q, kv, Hl, nope, rope, kvl, positions, table, kv_norm_w, eps, cache, slots, cu_q=None, vd=0, kv_lens=None):
    """What sits between the MLA projections and the MLA attention: split every query head of q [T, Hl*(nope+rope)]
    into its no-position part and its rotated part (interleaved pairs), RMS-normalise the compressed KV kv[:, :kvl],
    rotate the shared key part kv[:, kvl:], and append (normalised KV ‖ rotated key) to the latent cache at `slots`.
    Returns (q_nope [T,Hl,nope], q_rope [T,Hl,rope]).  One kernel on the GPU.  `cu_q` and `kv_lens` (prompts) and `vd`, the values' size:
    what the attention behind it is asked for, so that the queries come in the layout that it reads."""
    if _cuda(q) and cache.dtype == torch.bfloat16:
        from ..utils.flags import Env
        from .native_mla import expands
        return _nat().mla_prep(q, kv, Hl, nope, rope, kvl, positions, table, kv_norm_w, eps, cache, slots,
                               cu_q is not None and Env.get().mla_expand and expands(cu_q, nope, rope, kvl, vd, kv_lens))
    T = q.shape[0]
    q3 = q.reshape(T, Hl, nope + rope)
    ckv = R.rmsnorm(kv[:, :kvl], kv_norm_w, eps)
    q_rope, kr = R.rope_apply(q3[..., nope:], kv[:, kvl:].reshape(T, 1, rope), positions, table, rope, "interleaved", 0)
    latent_cache_write(torch.cat([ckv, kr.reshape(T, rope)], dim=-1), cache, slots)
    return q3[..., :nope].contiguous(), q_rope.contiguous()


@dataclass(frozen=True)
class LatentDims:
    """Sizes of a latent-attention layer as its kernels see them (heads of this rank; sizes possibly padded with zeros).
    A packed row is [q: heads x (dim + rot) | latent: rank + rot (unless the layer reads another's) | gate: heads x vdim], or
    with `head_gate` one gate value per head, in a row of a multiple of `align` values."""
    heads: int
    dim: int                    # unrotated query/key dimensions per head
    rot: int                    # rotated dimensions per head
    rank: int                   # latent
    vdim: int
    own_kv: bool
    gate: bool
    rank_real: int              # values of the latent that are not padding (the norm's count)
    head_gate: bool = False
    align: int = 1

    @property
    def q_width(self) -> int:
        return self.heads * (self.dim + self.rot)

    @property
    def gate_at(self) -> int:
        return self.q_width + (self.rank + self.rot if self.own_kv else 0)

    @property
    def row(self) -> int:
        n = self.gate_at + (0 if not self.gate else self.heads if self.head_gate else self.heads * self.vdim)
        return (n + self.align - 1) // self.align * self.align


def latent_prep(x, dims: LatentDims, positions, table, rot_dims, norm_w, eps, cache, slots):
    """What sits between the packed projection x [T, dims.row] of a latent-attention layer and its attention: rotates the
    rotated part of every query in place (interleaved pairs, the first `rot_dims`), and, for a layer with a cache of its
    own, appends [RMS-normed latent | rotated key part] to `cache` [blocks, 1, block, rank + rot] at `slots`."""
    if _cuda(x):
        return _nat_latent().latent_prep(x, dims, positions, table, rot_dims, norm_w, eps, cache, slots)
    d, T = dims, x.shape[0]
    q = x[:, :d.q_width].view(T, d.heads, d.dim + d.rot)
    kr = x[:, d.q_width + d.rank:d.q_width + d.rank + d.rot].reshape(T, 1, d.rot) if d.own_kv else None
    if table is not None and rot_dims > 0:
        qr, kr = R.rope_apply(q[..., d.dim:], kr, positions, table, rot_dims, "interleaved")
        q[..., d.dim:] = qr
    if d.own_kv:
        c = x[:, d.q_width:d.q_width + d.rank].float()
        n = c * torch.rsqrt(c.pow(2).sum(-1, keepdim=True) / d.rank_real + eps) * norm_w
        latent_cache_write(torch.cat([n.to(x.dtype), kr.reshape(T, d.rot)], -1), cache, slots)


def latent_attention(x, dims: LatentDims, cache, block_table, cu_q, kv_lens, weights, scale, window=0, meta=None, sinks=None):
    """Attention of the packed rows x (after `latent_prep`) over a latent cache -> [T, heads * vdim], multiplied with the
    sigmoid of the rows' gate.  `weights`: `LatentWeights`.  `window` and `sinks` as in `paged_attention`."""
    if _cuda(x):
        return _nat_latent().latent_attention(x, dims, cache, block_table, cu_q, kv_lens, weights, scale, window, meta, sinks)
    d, T = dims, x.shape[0]
    q = x[:, :d.q_width].view(T, d.heads, d.dim + d.rot)
    a = R.mla_attention(q[..., :d.dim], q[..., d.dim:], cache, block_table, cu_q, kv_lens, weights.uk, weights.uv, scale,
                        max(cu_q[i + 1] - cu_q[i] for i in range(len(kv_lens))) == 1, window, sinks).reshape(T, -1)
    if d.gate and d.head_gate:
        g = torch.sigmoid(x[:, d.gate_at:d.gate_at + d.heads].float())[:, :, None]
        a = (a.view(T, d.heads, d.vdim).float() * g).to(a.dtype).reshape(T, -1)
    elif d.gate:
        a = (a.float() * torch.sigmoid(x[:, d.gate_at:d.gate_at + d.heads * d.vdim].float())).to(a.dtype)
    return a


class LatentWeights:
    """The per-head matrices of a latent-attention layer: uk [heads, dim, rank], uv [heads, vdim, rank]."""

    def __init__(self, uk, uv):
        self.uk, self.uv = uk.contiguous(), uv.contiguous()
        self.cache: dict = {}               # layouts the kernels want, made once


# -- attention whose values are its keys ------------------------------------------------------
@dataclass
class HeadPrep:
    """What happens to the heads of a packed row [q: hq x dim | k: hkv x dim] between projection and cache: weights of the
    short convolution [taps, (hq + hkv) * dim] fp32 (None: none), gains of the norms per head (None: none).  Heads leave
    `padded` wide, zeros behind `dim`."""
    hq: int
    hkv: int
    dim: int
    padded: int
    conv: Optional[torch.Tensor]
    q_norm: Optional[torch.Tensor]
    k_norm: Optional[torch.Tensor]

    @property
    def taps(self) -> int:
        return 1 if self.conv is None else self.conv.shape[0]


def head_prep(x, prep: HeadPrep, eps, positions, table, rot_dims, kc, vc, slots, state, state_slots, cu_q, kv_lens, meta=None):
    """Causal convolution over time on every channel of q and k, RMS norm per head, rotation of the first `rot_dims`
    dimensions; appends k to `kc` and the keys as they left the convolution to `vc`, and returns q [T, hq, padded].
    `state` [slots, taps - 1, channels] holds the last inputs of each sequence's convolution, oldest first, and is moved on
    to the end of this call's tokens; what lies before a sequence's first token counts as zero."""
    impl = _native_linear().head_prep if _cuda(x) else R.head_prep
    return impl(x, prep, eps, positions, table, rot_dims, kc, vc, slots, state, state_slots, cu_q, kv_lens, meta)


# -- gated linear attention -------------------------------------------------------------------
@dataclass(frozen=True)
class LinearDims:
    """A packed row of a gated-linear-attention layer: [q: heads x dim | k | v: heads x vdim | g | a1: rank], each part
    starting at a multiple of `align` values."""
    heads: int
    dim: int
    vdim: int
    rank: int
    align: int = 1

    def up(self, n: int) -> int:
        return (n + self.align - 1) // self.align * self.align

    @property
    def k_at(self) -> int:
        return self.up(self.heads * self.dim)

    @property
    def v_at(self) -> int:
        return 2 * self.k_at

    @property
    def g_at(self) -> int:
        return self.v_at + self.up(self.heads * self.vdim)

    @property
    def a_at(self) -> int:
        return self.g_at + self.up(self.heads * self.vdim)


@dataclass
class LinearWeights:
    """Decay and output norm: the decay's second product a2 [heads * dim, rank (aligned)] and its bias, `tau`, the gain of
    the norm over a head's vdim outputs ([vdim], or [heads * vdim]).  `scale` of the queries (None: 1 / sqrt(dim)).  `bonus`
    [heads, dim]: the current token is read with this factor on its key instead of through the state, and decays are
    exp(-exp(z)).  `mult`: a factor of the result."""
    a2: torch.Tensor
    bias: torch.Tensor
    tau: float
    norm: torch.Tensor
    scale: Optional[float] = None
    bonus: Optional[torch.Tensor] = None
    mult: float = 1.0


def gated_linear(x, dims: LinearDims, w: LinearWeights, eps, state, state_slots, cu_q, kv_lens, meta=None, out=None):
    """Gated linear attention of packed rows x -> [T, heads * vdim (aligned)] (into `out` when given).  Per head, with z = W_a2 a1
    + bias and decay = sigmoid(z)^(1 / tau) per key channel: S <- diag(decay) S + k v^T and o = S^T (q * scale); the result is
    norm(o) * silu(g).  With a bonus u: decay = exp(-exp(z)), and o = (S + diag(u) k v^T)^T q is read before S moves on.
    `state` [slots, heads, dim, vdim] fp32 is carried on; a sequence's first token starts from zero."""
    impl = _native_linear().gated_linear if _cuda(x) else R.gated_linear
    return impl(x, dims, w, eps, state, state_slots, cu_q, kv_lens, meta, out)


def token_shift(x, mu, state, state_slots, cu_q, kv_lens, dtype, meta=None):
    """Mixes of every row with the row of the token before it: column part i of the result [T, n * width] is
    x + (previous x - x) * mu[i] (mu [n, width] fp32), the arithmetic in fp32.  `state` [slots, width] fp32 holds the last row of
    each sequence and is moved on; in front of a sequence's first token are zeros."""
    impl = _native_linear().token_shift if _cuda(x) else R.token_shift
    return impl(x, mu, state, state_slots, cu_q, kv_lens, dtype, meta)


# -- state-space recurrence ---------------------------------------------------------------------
@dataclass(frozen=True)
class StateDims:
    """A packed row of a state-space layer: [z: heads x vdim | x: heads x vdim, B, C: groups x state each | dt: heads]; the three
    parts start at multiples of `align` values, and x, B, C are one run of channels."""
    heads: int
    state: int
    vdim: int
    groups: int
    norm_groups: int
    taps: int
    align: int = 1

    def up(self, n: int) -> int:
        return (n + self.align - 1) // self.align * self.align

    @property
    def inner(self) -> int:
        return self.heads * self.vdim

    @property
    def channels(self) -> int:
        return self.inner + 2 * self.groups * self.state

    @property
    def x_at(self) -> int:
        return self.up(self.inner)

    @property
    def dt_at(self) -> int:
        return self.x_at + self.up(self.channels)

    @property
    def row(self) -> int:
        return self.dt_at + self.up(self.heads)


@dataclass
class StateWeights:
    """fp32: the convolution [taps, channels] and its bias, per head dt_bias, the decay's rate exp(A_log) and the skip's factor D,
    the gain of the output norm [heads * vdim]."""
    conv: torch.Tensor
    conv_bias: torch.Tensor
    dt_bias: torch.Tensor
    rate: torch.Tensor
    skip: torch.Tensor
    norm: torch.Tensor


def state_space(x, dims: StateDims, w: StateWeights, eps, state, conv_state, state_slots, cu_q, kv_lens, meta=None):
    """The mixer of a state-space layer between its two projections, packed rows x -> [T, heads * vdim (aligned)]: x, B and C
    through a causal convolution and silu, dt through softplus, then per head S <- exp(-rate dt) S + dt B x^T and
    y = S^T C + D x; y * silu(z) is normalised in `norm_groups` parts.  `state` [slots, heads, state, vdim] fp32 and `conv_state`
    [slots, taps - 1, channels] (None for one tap) are carried on; a sequence's first token starts from zero."""
    impl = _native_linear().state_space if _cuda(x) else R.state_space
    return impl(x, dims, w, eps, state, conv_state, state_slots, cu_q, kv_lens, meta)


# -- attention with mixed heads -----------------------------------------------------------------
@dataclass
class TalkingHeads:
    """Attention whose heads' weights are mixed.  A packed row is [q: hq x dim | k: hkv x dim | gate: hq x padded], each part starting
    at a multiple of `align` values; heads leave `padded` wide.  Gains of the norms over the whole projections [hq * dim] and
    [hkv * dim], the distance bias r1, r2 [hq], the mixing matrix talk [hq, hq], all fp32.  `mult`: a factor of the result."""
    hq: int
    hkv: int
    dim: int
    padded: int
    q_norm: torch.Tensor
    k_norm: torch.Tensor
    r1: torch.Tensor
    r2: torch.Tensor
    talk: torch.Tensor
    mult: float = 1.0
    align: int = 1

    def up(self, n: int) -> int:
        return (n + self.align - 1) // self.align * self.align

    @property
    def k_at(self) -> int:
        return self.up(self.hq * self.dim)

    @property
    def gate_at(self) -> int:
        return self.k_at + self.up(self.hkv * self.dim)

    @property
    def row(self) -> int:
        return self.gate_at + self.up(self.hq * self.padded)


def talking_prep(x, d: TalkingHeads, eps, kc, vc, slots):
    """RMS norms over all of a row's q and over all of its k; appends k to `kc` and k as it was before its norm to `vc`, and
    returns q [T, hq, padded]."""
    return (_native_talking() if _cuda(x) else R).talking_prep(x, d, eps, kc, vc, slots)


def talking_attention(q, x, d: TalkingHeads, kc, vc, block_table, cu_q, kv_lens, scale, window=0, meta=None, out=None):
    """Attention with scores q . k * scale - r1 ln(1 + r2 (i - j)) over the keys that `window` leaves, a softmax per head, the heads'
    weights mixed by `talk` (head h applies sum_g talk[h, g] weight_g to the values of its own key/value head), and the gate of
    the packed rows x: -> [T, hq * padded] (into `out` when given)."""
    impl = (_native_talking() if _cuda(q) else R).talking_attention
    return impl(q, x, d, kc, vc, block_table, cu_q, kv_lens, scale, window, meta, out)


def _native_talking():
    from . import native_talking
    return native_talking


def _native_linear():
    from . import native_linear
    return native_linear


# -- MoE -----------------------------------------------------------------------------------
def route(logits, kind, top_k, bias=None, n_group=1, topk_group=1, routed_scaling=1.0, norm_topk=True,
          scoring="sigmoid"):
    if _cuda(logits):
        return _nat().route(logits, kind, top_k, bias, n_group, topk_group, routed_scaling, norm_topk, scoring)
    if kind == "mixtral":
        return R.route_mixtral(logits, top_k)
    if kind == "softmax_topk":
        return R.route_softmax_topk(logits, top_k, norm_topk)
    if kind == "deepseek":
        return R.route_deepseek(logits, bias, top_k, n_group, topk_group, routed_scaling, norm_topk, scoring)
    raise ValueError(kind)


def moe_experts(x, idx, w, experts, act="silu", expert_offset=0, packed=None, expected_pairs=None, gated=True, add=None):
    """Weighted sum of the chosen experts' outputs (see `reference.moe_experts`) in fp32, plus `add` [T, H] fp32."""
    if gated and experts and experts[0][0].kind == "fp8a":
        return moe_experts_e4m3(quantize_e4m3(x), idx, w, experts, act, expert_offset, packed, expected_pairs, add)
    if _cuda(x):
        return _nat().moe_experts(x, idx, w, experts, act, expert_offset, packed, expected_pairs, gated, add)
    out = R.moe_experts(x, idx, w, experts, act, expert_offset, gated)
    return out if add is None else out + add


# -- sampling ------------------------------------------------------------------------------
def argmax_rows(logits):
    if _cuda(logits):
        return _nat().argmax_rows(logits)
    return R.argmax_rows(logits)


def beam_topk(logits, k):
    """(log-softmax values, token ids) of each row's k best entries, best first."""
    if _cuda(logits):
        from . import native_sample
        return native_sample.beam_topk(logits, k)
    return R.beam_topk(logits, k)


def sample_top_k_top_p(logits, top_k, top_p, temperature, uniform):
    if _cuda(logits):
        return _nat().sample_top_k_top_p(logits, top_k, top_p, temperature, uniform)
    return R.sample_top_k_top_p(logits, top_k, top_p, temperature, uniform)
