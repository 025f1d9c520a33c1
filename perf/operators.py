"""What the operators of the block-scaled 8-bit path are measured on: rows in e4m3 with a scale for each 128 columns.

A layer whose weights and activations are e4m3 is made of four of them, each case is one call of one:

* ``norm``      the residual's addition, RMSNorm and quantisation of its output in one (`ops.rmsnorm_e4m3`)
* ``linear``    a product of e4m3 rows with e4m3 weights, a scale for each 128 columns of a row and each 128 x 128 block of the
                weights (`ops.linear_e4m3`)
* ``gated``     act(gate) * up of two such products, quantised for the next one (`ops.linear_gated_e4m3`)
* ``experts``   the routed experts' gated and down products and their weighted sum (`ops.moe_experts_e4m3`)

A row's values y in a block of 128 columns become codes e4m3(y * (448 / a)) and the scale a / 448, a = max |y| (at least 2^-100).
Scales lie block by block, [blocks, rows]; a product's weights are [features, columns].
"""
import math

import torch

own = False

_BLOCK = 128
_TOP = 448.0
_LEAST = 2.0 ** -100
_EPS = 1e-6
_E4M3 = torch.float8_e4m3fn


def _norm(T, K, residual, rows, name=None):
    c = {"op": "norm", "T": T, "K": K, "residual": residual, "rows": rows}
    return dict(c, name=name) if name else c


def _linear(T, N, K, bias=False, residual=False, out="bf16", name=None):
    c = {"op": "linear", "T": T, "N": N, "K": K, "bias": bias, "residual": residual, "out": out}
    return dict(c, name=name) if name else c


def _gated(T, I, K, name=None):
    c = {"op": "gated", "T": T, "I": I, "K": K}
    return dict(c, name=name) if name else c


def _experts(T, E, k, H, I, name=None):
    c = {"op": "experts", "T": T, "E": E, "k": k, "H": H, "I": I}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's step: the norm in front of a product, nothing but latency
        _norm(1, 4096, "none", False, "norm-1"),
        # between expert layers: the experts' sum in 32 bits joins the stream, the router wants the rows in bf16 too; odd row count
        _norm(777, 7168, "fp32", True, "norm-experts"),
        # a pass of prompts of a wide model, the sublayer's output in bf16
        _norm(16384, 8192, "bf16", False, "norm-prompt"),
        # one user's step: the projection to queries, keys and values
        _linear(1, 12288, 4096, name="qkv-1"),
        # a batch of decode steps: output projection, long rows, the residual in the epilogue, one row past a tile
        _linear(33, 7168, 16384, residual=True, name="o-33"),
        # a short prompt: the merged down-projection of latent attention, features that end inside a block of scales
        _linear(389, 2112, 7168, name="latent-389"),
        # a pass of prompts of a wide model: the second product of the feed-forward
        _linear(8192, 8192, 28672, residual=True, name="down-prompt"),
        # feed-forward of a decode step, and of a pass of prompts
        _gated(16, 11008, 4096, "gated-16"),
        _gated(4096, 14336, 4096, "gated-prompt"),
        # narrow experts: a few users' step and a pass of prompts
        _experts(8, 64, 6, 2048, 1408, "experts-8"),
        _experts(4096, 64, 6, 2048, 1408, "experts-prompt"),
        # wide experts, a batch of short prompts
        _experts(300, 8, 2, 4096, 14336, "experts-wide"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "gated", "experts"])
    if op == "norm":
        K = 8 * _log(rng, 32, 2048)
        return _norm(_log(rng, 1, min(16384, 16384 * 8192 // K)), K, rng.choice(["none", "bf16", "fp32"]), rng.random() < 0.4)
    if op == "linear":
        K = 8 * _log(rng, 16, 3584)
        N = _log(rng, 32, min(57344, 28672 * 8192 // K))
        T = _log(rng, 1, min(8192, 8192 * 8192 * 28672 // (N * K)))
        return _linear(T, N, K, rng.random() < 0.3, rng.random() < 0.5, rng.choice(["bf16", "bf16", "fp32"]))
    if op == "gated":
        K, I = 16 * _log(rng, 16, 512), _BLOCK * _log(rng, 1, 224)
        return _gated(_log(rng, 1, min(8192, 4096 * 8192 * 28672 // (I * K))), I, K)
    H, I, E = _BLOCK * _log(rng, 4, 56), _BLOCK * _log(rng, 2, 112), _log(rng, 2, 64)
    E = max(2, min(E, 64 * 2048 * 1408 * 2 // (H * I)))
    return _experts(_log(rng, 1, max(2, min(4096, 4096 * 64 * 2048 * 1408 // (E * H * I)))), E, rng.randint(1, min(8, E)), H, I)


# -- inputs ---------------------------------------------------------------------------------------------------------
def _activations(g, T, K):
    """Rows as a trained model has them: channels of very different size, a few of them far above the others."""
    channel = torch.exp(0.5 * torch.randn(K, generator=g, device="cuda"))
    channel = torch.where(torch.rand(K, generator=g, device="cuda") < 0.005, 20 * channel, channel)
    return (torch.randn(T, K, generator=g, device="cuda") * channel).bfloat16()


def _row_codes(x):
    """(codes [T, K], scales [blocks, T]) of rows."""
    T, K = x.shape
    n = -(-K // _BLOCK)
    y = torch.nn.functional.pad(x.float(), (0, n * _BLOCK - K)).view(T, n, _BLOCK)
    a = y.abs().amax(-1).clamp_min(_LEAST)
    return (y * (_TOP / a)[..., None]).view(T, -1)[:, :K].to(_E4M3).contiguous(), (a / _TOP).t().contiguous()


def _weights(g, N, K, lead=()):
    """(codes [*lead, N, K], scales [*lead, blocks of N, blocks of K]) of weights around zero, rows of different size."""
    n, m = -(-N // _BLOCK), -(-K // _BLOCK)
    w = torch.zeros(*lead, n * _BLOCK, m * _BLOCK, device="cuda", dtype=torch.bfloat16)
    w[..., :N, :K] = torch.randn(*lead, N, K, generator=g, device="cuda", dtype=torch.bfloat16)
    w *= (K ** -0.5 * torch.exp(0.3 * torch.randn(*lead, n * _BLOCK, 1, generator=g, device="cuda"))).bfloat16()
    b = w.view(*lead, n, _BLOCK, m, _BLOCK)
    s = b.abs().amax(dim=(-3, -1)).float() / _TOP
    q = (b / s[..., :, None, :, None].bfloat16()).view(*lead, n * _BLOCK, m * _BLOCK)
    return q[..., :N, :K].clamp(-_TOP, _TOP).to(_E4M3).contiguous(), s.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    s = dict(case)
    if case["op"] == "norm":
        T, K = case["T"], case["K"]
        s["x"], s["gain"] = _activations(g, T, K), 1 + 0.2 * randn(K)
        s["r"] = None if case["residual"] == "none" else randn(T, K).to(torch.float32 if case["residual"] == "fp32" else torch.bfloat16)
    elif case["op"] == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        s["q"], s["sx"] = _row_codes(_activations(g, T, K))
        s["w"], s["sw"] = _weights(g, N, K)
        s["bias"] = randn(N) if case["bias"] else None
        s["r"] = randn(T, N).bfloat16() if case["residual"] else None
    elif case["op"] == "gated":
        s["q"], s["sx"] = _row_codes(_activations(g, case["T"], case["K"]))
        s["w"], s["sw"] = _weights(g, 2 * case["I"], case["K"])
    else:
        T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
        s["q"], s["sx"] = _row_codes(_activations(g, T, H))
        s["gu"], s["gus"] = _weights(g, 2 * I, H, (E,))
        s["dn"], s["dns"] = _weights(g, H, I, (E,))
        score = randn(T, E) + 0.7 * randn(E)                             # some experts are asked for more often
        top, idx = score.topk(k, dim=1)
        s["idx"], s["wt"] = idx.int(), torch.softmax(top, 1)
    if own:                                                              # the handles that a program holds: weights as the loader makes
        from xfastertransformer_b200 import ops                          # them, rows as the product before left them
        from xfastertransformer_b200.runtime.loader import make_linear
        if "q" in s:
            s["rows_in"] = ops.RowsE4M3(s["q"], s["sx"])
        if "w" in s:
            s["W"] = make_linear(s["w"], "fp8a", scale=s["sw"])
        if "gu" in s:
            s["experts"] = [(make_linear(s["gu"][e], "fp8a", scale=s["gus"][e]), make_linear(s["dn"][e], "fp8a", scale=s["dns"][e]))
                            for e in range(case["E"])]
            s["packed"] = ops.pack_experts_e4m3(s["experts"])
            del s["gu"], s["gus"], s["dn"], s["dns"]                     # the experts' codes are held once
    return s


# -- plain form -----------------------------------------------------------------------------------------------------
def _values(q, sx):
    return q.float() * sx.t().repeat_interleave(_BLOCK, 1)[:, :q.shape[1]]


def _dense(w, sw):
    s = sw.repeat_interleave(_BLOCK, -2)[..., :w.shape[-2], :].repeat_interleave(_BLOCK, -1)[..., :w.shape[-1]]
    return w.float() * s


def _coded(y):
    """(codes, scales [blocks, ...]) of fp32 rows [..., K]."""
    K = y.shape[-1]
    n = -(-K // _BLOCK)
    b = torch.nn.functional.pad(y, (0, n * _BLOCK - K)).view(*y.shape[:-1], n, _BLOCK)
    a = b.abs().amax(-1).clamp_min(_LEAST)
    q = (b * (_TOP / a)[..., None]).reshape(*y.shape[:-1], n * _BLOCK)[..., :K].to(_E4M3)
    return q.contiguous(), (a / _TOP).movedim(-1, 0).contiguous()


def _plain(s):
    op = s["op"]
    if op == "norm":
        h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).bfloat16()
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS) * s["gain"]
        q, scale = _coded(y)
        return q, scale, y.bfloat16() if s["rows"] else None, None if s["r"] is None else h
    x = _values(s["q"], s["sx"])
    if op == "linear":
        y = x @ _dense(s["w"], s["sw"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["r"] is not None:
            y = y + s["r"].float()
        return y if s["out"] == "fp32" else y.bfloat16()
    if op == "gated":
        y = x @ _dense(s["w"], s["sw"]).t()
        gate, up = y[:, :s["I"]], y[:, s["I"]:]
        return _coded(gate / (1 + torch.exp(-gate)) * up)
    # every expert for every token, and the sum weighted with what the tokens chose
    y = x[None] @ _dense(s["gu"], s["gus"]).transpose(1, 2)
    gate, up = y[..., :s["I"]], y[..., s["I"]:]
    q, scale = _coded(gate / (1 + torch.exp(-gate)) * up)
    del y, gate, up
    v = q.float() * scale.movedim(0, -1).repeat_interleave(_BLOCK, -1)
    z = v @ _dense(s["dn"], s["dns"]).transpose(1, 2)
    share = torch.zeros(s["T"], s["E"], device=x.device).scatter_(1, s["idx"].long(), s["wt"])
    return (z * share.t()[:, :, None]).sum(0).bfloat16()


# -- the framework's ------------------------------------------------------------------------------------------------
def _calls(s):
    from xfastertransformer_b200 import ops
    op = s["op"]
    if op == "norm":
        q, y, h = ops.rmsnorm_e4m3(s["x"], s["gain"], _EPS, residual=s["r"], want_rows=s["rows"])
        return q.codes, q.scale, y, h
    if op == "linear":
        return ops.linear_e4m3(s["rows_in"], s["W"], s["bias"], residual=s["r"], out_dtype=torch.float32 if s["out"] == "fp32" else torch.bfloat16)
    if op == "gated":
        q = ops.linear_gated_e4m3(s["rows_in"], s["W"], "silu")
        return q.codes, q.scale
    return ops.moe_experts_e4m3(s["rows_in"], s["idx"], s["wt"], s["experts"], "silu", packed=s["packed"], out_dtype=torch.bfloat16)


def run(state):
    return _calls(state) if own else _plain(state)


# -- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    up = lambda n: -(-n // _BLOCK)
    T = case["T"]
    if case["op"] == "norm":
        K = case["K"]
        r = {"none": 0, "bf16": 2 + 2, "fp32": 4 + 2}[case["residual"]]       # what is added, and the stream that goes on
        return {"bytes": T * K * (2 + 1 + r + (2 if case["rows"] else 0)) + 4 * T * up(K) + 4 * K, "flops": 10.0 * T * K}
    if case["op"] == "linear":
        N, K = case["N"], case["K"]
        out = (4 if case["out"] == "fp32" else 2) + (2 if case["residual"] else 0)
        return {"bytes": N * K + T * K + 4 * up(K) * (up(N) + T) + T * N * out + (4 * N if case["bias"] else 0), "flops": 2.0 * T * N * K}
    if case["op"] == "gated":
        I, K = case["I"], case["K"]
        return {"bytes": 2 * I * K + T * K + 4 * up(K) * (2 * up(I) + T) + T * I + 4 * T * up(I), "flops": 4.0 * T * I * K}
    E, k, H, I = (case[n] for n in ("E", "k", "H", "I"))
    asked = E * (1 - (1 - k / E) ** T)                                        # experts that some token chose
    return {"bytes": asked * 3 * H * I + T * H + 4 * T * up(H) + T * k * 8 + 2 * T * H, "flops": 6.0 * T * k * H * I}


# -- in 64 bits -----------------------------------------------------------------------------------------------------
def _exact_rows(v):
    """Codes and scales of rows in fp64, block after block."""
    codes, scales = torch.empty(v.shape, dtype=_E4M3, device=v.device), []
    for at in range(0, v.shape[1], _BLOCK):
        part = v[:, at:at + _BLOCK]
        top = torch.maximum(part.max(1).values, -part.min(1).values).clamp(min=_LEAST)
        codes[:, at:at + _BLOCK] = (part * _TOP / top[:, None]).to(_E4M3)
        scales.append(top / _TOP)
    return codes, torch.stack(scales)


def _exact_product(q, sx, w, sw):
    """sum over blocks of k: scales times the codes' product, in fp64."""
    a = q.double()
    b = w.double()
    for j in range(sx.shape[0]):
        at = slice(j * _BLOCK, (j + 1) * _BLOCK)
        a[:, at] *= sx[j].double()[:, None]
        b[:, at] *= sw[:, j].double().repeat_interleave(_BLOCK)[:w.shape[0], None]
    return torch.matmul(a, b.T)


def _exact_gated(q, sx, w, sw):
    both = _exact_product(q, sx, w, sw)
    g, u = both.chunk(2, dim=1)
    return _exact_rows(torch.sigmoid(g) * g * u)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "norm":
        x = s["x"]
        stream = None
        if s["r"] is not None:
            stream = (s["x"].double() + s["r"].double()).bfloat16()       # the sum rounds once, to the stream's type
            x = stream
        d = x.double()
        rms = torch.sqrt(torch.mean(torch.square(d), dim=1) + _EPS)
        v = d / rms[:, None] * s["gain"].double()[None]
        codes, scales = _exact_rows(v)
        return codes, scales, v if case["rows"] else None, stream
    if case["op"] == "linear":
        y = _exact_product(s["q"], s["sx"], s["w"], s["sw"])
        y = y if s["bias"] is None else y + s["bias"].double()
        return y if s["r"] is None else y + s["r"].double()
    if case["op"] == "gated":
        return _exact_gated(s["q"], s["sx"], s["w"], s["sw"])
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        token, slot = torch.nonzero(s["idx"] == e, as_tuple=True)
        if token.numel():
            q, sx = _exact_gated(s["q"][token], s["sx"][:, token], s["gu"][e], s["gus"][e])
            y = _exact_product(q, sx, s["dn"][e], s["dns"][e])
            out[token] += y * s["wt"][token, slot].double()[:, None]
    return out
