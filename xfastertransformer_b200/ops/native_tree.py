"""Bindings of the kernels for a step with trees of drafted tokens: masks and accepted paths (csrc/kernels/tree.cu), attention over
the paged cache (csrc/kernels/tree_attention.cu), sampling with every row's own limits (csrc/kernels/sample_rows.cu).

Nothing here keeps scratch between calls, so calls on several streams and captured graphs do not touch one another; the kernels run on
the device of their rows, on that device's current stream."""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from . import native as N


# csrc/kernels/tree.cu:TreeMaskArgs: cu_q, kv_lens | B, T | parents, mask, positions, status | words
MASK_ARGS = struct.Struct("@2P2i4Pi4x")
# csrc/kernels/tree.cu:TreeAcceptArgs: cu_q, kv_lens | B, T | tokens, sampled, parents, table, pools, emitted, path, count, status |
# table_ld | table_w, n_pools, bs, num_blocks, width
ACCEPT_ARGS = struct.Struct("@2P2i9Pq5i4x")
# csrc/kernels/tree_attention.cuh:TreeAttnArgs: q, out, kc, vc, ks, vs, table, cu_q, kv_lens, mask, positions, sinks, part_o, part_ml, status |
# table_ld | B, T, max_q, hq, hkv, group, q_off, D, bs, num_blocks, table_w, words, nsplit, window, keep | scale, softcap | form
ATTN_ARGS = struct.Struct("@15Pq15i2fi")
# csrc/kernels/sample_rows.cu:SampleArgs: x, temperature, top_k, top_p, min_p, uniform, out | ld | rows, V, bf16, k0 | t0, p0, m0
SAMPLE_ARGS = struct.Struct("@7Pq4i3f4x")
_P, _I = C.c_void_p, C.c_int
_ARGS = {"xft_tree_mask": [C.c_char_p, _I, _P], "xft_tree_accept": [C.c_char_p, _P], "xft_tree_attention": [C.c_char_p, _P],
         "xft_sample_rows": [C.c_char_p, _P]}
_fns = None


def _lib():
    global _fns
    if _fns is None:
        lib = N.lib()
        for name, args in _ARGS.items():
            f = getattr(lib, name)
            f.restype, f.argtypes = _I, args
        _fns = lib
    return _fns


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _foreign(device) -> bool:
    """Whether `device` is another than the current one, which allocations, stream and launches would go to."""
    return device.index != torch._C._cuda_getDevice()


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _i32(t):
    """Parents as the kernels take them: of int64 ones, those beyond 32 bits stay below zero or behind every node."""
    return t.contiguous() if t.dtype is torch.int32 else t.clamp(-1, 2 ** 31 - 1).int().contiguous()


def _arrays(cu_q, kv_lens, meta, dev):
    """(cu_q, kv_lens on the device, sequences, most nodes of one, longest cache)."""
    if meta is not None and getattr(meta, "cu_q_dev", None) is not None:
        cu, kv = meta.cu_q_dev, meta.kv_lens_dev
        if meta.max_q and meta.max_kv:
            return cu, kv, kv.numel(), meta.max_q, meta.max_kv
    else:
        cu = torch.tensor(list(cu_q), dtype=torch.int32, device=dev)
        kv = torch.tensor(list(kv_lens), dtype=torch.int32, device=dev)
    n = [b - a for a, b in zip(cu_q, cu_q[1:])]
    return cu, kv, kv.numel(), max(n, default=0), max(kv_lens, default=0)


MAX_SEQUENCES = 65535                # of one launch: the grid has a row of CTAs for each


def _few(what, B):
    if B > MAX_SEQUENCES:
        raise N.KernelError(f"{what}: up to {MAX_SEQUENCES} sequences at a time, not {B}")


def _padded(cu_q, T) -> bool:
    """Whether there are rows in front of the first sequence or behind the last one."""
    return isinstance(cu_q, (list, tuple)) and len(cu_q) > 0 and (cu_q[0] > 0 or cu_q[-1] < T)


def tree_mask(parents, cu_q, kv_lens, meta=None):
    dev = parents.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return tree_mask(parents, cu_q, kv_lens, meta)
    parents = _i32(parents)
    cu, kv, B, most, _ = _arrays(cu_q, kv_lens, meta, dev)
    T, words = parents.numel(), max(1, -(-most // 64))
    if _padded(cu_q, T):
        mask, positions = parents.new_zeros((T, words), dtype=torch.int64), torch.zeros_like(parents)
    else:
        mask, positions = parents.new_empty((T, words), dtype=torch.int64), torch.empty_like(parents)
    if T and B and most:
        ws = N.Workspace.get(dev)
        a = MASK_ARGS.pack(cu.data_ptr(), kv.data_ptr(), B, T, parents.data_ptr(), mask.data_ptr(), positions.data_ptr(), ws.status.data_ptr(),
                           words)
        rc = _lib().xft_tree_mask(a, most, _stream())
        if rc:
            N._check(rc, "tree_mask")
        ws.launches += 1
    return mask, positions


def _plan(B, hkv, rows, total, D, max_kv, tensor, int8=False):
    """(form, slices that the keys are cut into): the kernel of csrc/kernels/tree_attention_sm100.cu with one tile of 128 rows per CTA or
    (int8: codes are expanded once for both) two, or (form 0) that of tree_attention.cu.  `rows` over a key, `total` of all sequences and heads."""
    form = 0 if not tensor else 2 if int8 and rows > 128 else 1
    tall, slots = (64, 296) if not form else (128 * form, 148 if int8 or D == 256 else 296)
    ctas = B * hkv * -(-rows // tall)
    tiles = -(-max_kv // 128)
    most = max(1, min(tiles // (1 if form else 2), 64))
    best = None
    # slices that fill the SMs by half, once, twice, ...  us: a tile of 128 keys in a CTA that is alone on its SM, or one of two; a CTA's start
    # and end 3; the second launch 2.5, and 0.27 ns for each row and slice that it joins
    one, two = (3.0, 3.0) if int8 or not form else (1.4, 1.7) if D == 64 else (2.0, 2.8) if D == 128 else (2.6, 2.6)
    for k in (0.5, 1, 2, 3):
        n = max(1, min(int(k * slots) // ctas, most))
        cost = -(-ctas * n // slots) * (-(-tiles // n) * (one if ctas * n <= 148 else two) + 3) + (2.5 + 2.7e-4 * total * n if n > 1 else 0)
        if best is None or cost < best[0]:
            best = cost, n
    return form, best[1]


def tree_attention(q, kc, vc, block_table, cu_q, kv_lens, mask, scale, ks=None, vs=None, group=1, q_off=0, meta=None, softcap=0.0, window=0,
                   keep_first=0, sinks=None, positions=None):
    dev = q.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return tree_attention(q, kc, vc, block_table, cu_q, kv_lens, mask, scale, ks, vs, group, q_off, meta, softcap, window, keep_first,
                                  sinks, positions)
    T, hq, D = q.shape
    nb, hkv, bs, _ = kc.shape
    if q.dtype is not torch.bfloat16 or D not in (64, 128, 256) or kc.dtype is not (torch.bfloat16 if ks is None else torch.int8):
        raise N.KernelError(f"tree_attention: bf16 queries over a bf16 or int8 cache with heads of 64, 128 or 256, not {q.dtype} over {kc.dtype} "
                            f"with {D}")
    if (kc.data_ptr() | vc.data_ptr()) % 16:
        raise N.KernelError("tree_attention: caches start on 16 bytes")
    q = q if q.is_contiguous() and q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
    mask = mask if mask.is_contiguous() else mask.contiguous()
    block_table = block_table if block_table.stride(1) == 1 else block_table.contiguous()
    cu, kv, B, most, longest = _arrays(cu_q, kv_lens, meta, dev)
    out = torch.zeros_like(q) if _padded(cu_q, T) else torch.empty_like(q)
    if not (T and hq and B and most):
        return out
    _few("tree_attention", B)
    ws = N.Workspace.get(dev)
    form, n = _plan(B, hkv, most * group, T * hq, D, min(longest, window + keep_first + most + 256) if window else longest,
                    (D == 128 or ks is None) and bs % 64 == 0 and (scale > 0 or softcap > 0) and nb * hkv * bs < 2 ** 31 and (_ptr(ks) | _ptr(vs)) % 16 == 0,
                    ks is not None)
    part = q.new_empty(T * hq * n * (D + 2), dtype=torch.float32) if n > 1 else None
    po = _ptr(part)
    a = ATTN_ARGS.pack(q.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(), _ptr(ks), _ptr(vs), block_table.data_ptr(), cu.data_ptr(),
                       kv.data_ptr(), mask.data_ptr(), _ptr(positions), _ptr(sinks), po, po + T * hq * n * D * 4, ws.status.data_ptr(),
                       block_table.stride(0), B, T, most, hq, hkv, group, q_off, D, bs, nb, block_table.shape[1], mask.shape[1], n, min(window, 1 << 30),
                       min(keep_first, 1 << 30), scale, softcap, form)
    rc = _lib().xft_tree_attention(a, _stream())
    if rc:
        N._check(rc, "tree_attention")
    ws.launches += 2 if n > 1 else 1
    return out


def _per_row(v, rows, dtype, dev):
    """(tensor or None, number): a parameter of every row, or one for all."""
    if not isinstance(v, torch.Tensor):
        return None, v if dtype is torch.int32 or not abs(v) > 3.4e38 else math.copysign(math.inf, v)
    if v.dtype is dtype and v.numel() == rows and v.device == dev and v.is_contiguous():
        return v, 0
    if v.numel() == 1 and rows != 1:
        v = v.reshape(1).expand(rows)
    if dtype is torch.int32 and v.dtype is torch.int64:                 # (beyond 32 bits: as good as none, and not the low 32 bits)
        v = v.clamp(-1, 2 ** 31 - 1)
    return v.to(device=dev, dtype=dtype).contiguous(), 0


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    dev = logits.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return sample(logits, temperature, top_k, top_p, min_p, uniform)
    V = logits.shape[-1]
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.dtype is not torch.float32 and x.dtype is not torch.bfloat16:
        x = x.float()
    if x.stride(1) != 1 and V > 1:
        x = x.contiguous()
    rows = x.shape[0]
    out = x.new_empty(rows, dtype=torch.int64)
    if rows:
        t, t0 = _per_row(temperature, rows, torch.float32, dev)
        k, k0 = _per_row(top_k, rows, torch.int32, dev)
        p, p0 = _per_row(top_p, rows, torch.float32, dev)
        m, m0 = _per_row(min_p, rows, torch.float32, dev)
        u, _ = _per_row(uniform, rows, torch.float32, dev)
        a = SAMPLE_ARGS.pack(x.data_ptr(), _ptr(t), _ptr(k), _ptr(p), _ptr(m), u.data_ptr(), out.data_ptr(), x.stride(0), rows, V,
                             x.dtype is torch.bfloat16, max(-1, min(int(k0), 2 ** 31 - 1)), t0, p0, m0)
        rc = _lib().xft_sample_rows(a, _stream())
        if rc:
            N._check(rc, "sample")
        N.Workspace.get(dev).launches += 1
    return out if logits.dim() == 2 else out.view(logits.shape[:-1])


class CachePools:
    """Where the pools of all layers are, for `tree_accept`: rows [address, heads, bytes of a head's row] on their device.  Holds the pools."""

    def __init__(self, pools):
        self.pools = pools
        first = pools[0]
        self.num_blocks, self.block = first.shape[0], first.shape[2]
        self.table = torch.tensor([[p.data_ptr(), p.shape[1], p.element_size() * (p.shape[3] if p.dim() == 4 else 1)] for p in pools],
                                  dtype=torch.int64).to(first.device)
        if first.is_cuda:
            torch.cuda.current_stream(first.device).synchronize()       # other streams may read it from now on
        self.retired = False

    def retire(self):
        """The pools are replaced: lets them go.  `tree_accept` refuses the handle from now on, and a graph captured with it moves nothing."""
        self.retired, self.pools = True, []
        self.table[:, 1:].zero_()                                        # no heads, rows of no bytes (a launch under way may still use an address)


def tree_accept(tokens, parents, sampled, cu_q, kv_lens, block_table, pools, meta=None):
    dev = tokens.device
    if _foreign(dev):
        with torch.cuda.device(dev):
            return tree_accept(tokens, parents, sampled, cu_q, kv_lens, block_table, pools, meta)
    parents = _i32(parents)
    tokens, sampled = (t if t.dtype is torch.int64 and t.is_contiguous() else t.long().contiguous() for t in (tokens, sampled))
    cu, kv, B, most, _ = _arrays(cu_q, kv_lens, meta, dev)
    _few("tree_accept", B)
    T = tokens.numel()
    emitted, path, count = tokens.new_empty((B, most)), parents.new_empty((B, most)), parents.new_empty(B)
    if B and most:
        if block_table is not None and block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        ws = N.Workspace.get(dev)
        a = ACCEPT_ARGS.pack(cu.data_ptr(), kv.data_ptr(), B, T, tokens.data_ptr(), sampled.data_ptr(), parents.data_ptr(), _ptr(block_table),
                             0 if pools is None else pools.table.data_ptr(), emitted.data_ptr(), path.data_ptr(), count.data_ptr(),
                             ws.status.data_ptr(), 0 if block_table is None else block_table.stride(0),
                             0 if block_table is None else block_table.shape[1], 0 if pools is None else len(pools.pools),
                             0 if pools is None else pools.block, 0 if pools is None else pools.num_blocks, most)
        rc = _lib().xft_tree_accept(a, _stream())
        if rc:
            N._check(rc, "tree_accept")
        ws.launches += 1
    else:
        count.zero_()
    return emitted, path, count
