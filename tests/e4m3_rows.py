"""What the tests of the block-scaled e4m3 operators share: inputs and their formulas in 64 bits."""
import torch

from xfastertransformer_b200 import ops
from xfastertransformer_b200.runtime.loader import LinearWeight, make_linear

TOP, LEAST = 448.0, 2.0 ** -100


def gen(*seed):
    return torch.Generator(device="cpu").manual_seed(sum(int(s) * p for s, p in zip(seed, (1, 7, 31, 101, 1009))))


def activations(g, T, K, dtype=torch.bfloat16):
    """Channels of different size, one of them far above the others, and rows from one end of the type to the other."""
    x = torch.randn(T, K, generator=g) * torch.exp(torch.randn(K, generator=g))
    x[:, K // 3] *= 50
    if T > 3:
        x[1], x[2] = x[1] * 1e-20, x[2] * 1e20
    return x.to(dtype)


def weight(g, N, K, kind="fp8a", std=0.05):
    w = torch.randn(N, K, generator=g) * std * torch.exp(0.5 * torch.randn(N, 1, generator=g))
    return make_linear(w, kind)


def scaled(W, scale):
    """The weight with other scales."""
    return LinearWeight(W.kind, W.w, scale, block=W.block, in_features=W.in_features, out_features=W.out_features)


def rows(x):
    return ops.quantize_e4m3(x)


def on(W, device="cuda"):
    return W.to(device)


def rows_on(q, device="cuda"):
    return ops.RowsE4M3(q.codes.to(device), q.scale.to(device))


def values64(q):
    K = q.codes.shape[1]
    return q.codes.cpu().double() * q.scale.cpu().double().t().repeat_interleave(128, 1)[:, :K]


def dense64(W):
    o, i = W.w.shape
    s = W.scale.cpu().double().repeat_interleave(128, 0)[:o].repeat_interleave(128, 1)[:, :i]
    return W.w.cpu().double() * s


def sum_tol(q, W):
    """(product in 64 bits, how far an fp32 product may be off).  The 128 products of a block are exact in fp32; each of the 128 additions
    and of the two roundings per block's scaling and addition is off by at most 2^-24 of the sum of magnitudes (the tensor core, which cuts
    instead of rounding, by 2^-23 for each of the 4 steps of a block)."""
    x, w = values64(q), dense64(W)
    mag = x.abs() @ w.abs().t()
    blocks = q.scale.shape[0]
    return x @ w.t(), (128 + 8 + 3 * blocks) * 2.0 ** -24 * mag


def coded_error(got, want, err):
    """Largest (|got - want| - allowed) of rows in e4m3 against fp64 rows `want` that were known to `err` when they were quantised: half a step
    of e4m3, relative 2^-4 and 2^-10 of the scale below its normal numbers, 2^-20 for the factor and the scale in fp32."""
    v = values64(got)
    s = got.scale.cpu().double().t().repeat_interleave(128, 1)[:, :v.shape[1]]
    half = torch.maximum(2.0 ** -4 * (want.abs() + err), 2.0 ** -10 * s)
    return ((v - want).abs() - (half * (1 + 2.0 ** -10) + err + 2.0 ** -20 * want.abs())).max().item()


def scale_error(got, want, err):
    """The same of the scales: a / 448 with a known to the block's largest `err`."""
    K = want.shape[1]
    pad = lambda t: torch.nn.functional.pad(t, (0, -K % 128)).view(t.shape[0], -1, 128).amax(-1).t()
    a, e = pad(want.abs()).clamp_min(LEAST), pad(err)
    return ((got.scale.cpu().double() * TOP - a).abs() - (e + 2.0 ** -22 * a)).max().item()
