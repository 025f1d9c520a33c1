"""Rows in e4m3 and their products on a CPU: the formulas against 64 bits, refusals, the parameter struct, and models of dtype "fp8_w8a8"."""
import ctypes as C

import pytest
import torch

import xfastertransformer_b200 as xft
from e4m3_rows import activations, coded_error, gen, rows, scale_error, scaled, sum_tol, values64, weight
from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import reference as R
from xfastertransformer_b200.config import ModelConfig, RopeConfig
from xfastertransformer_b200.runtime.loader import LinearWeight, cat_linear, make_linear
from xfastertransformer_b200.tools.synthetic import preset, write_synthetic_checkpoint
from xfastertransformer_b200.utils.flags import Env


@pytest.mark.parametrize("T,K", [(1, 1), (3, 128), (5, 200), (4, 1032)])
def test_rows_stand_for_their_values(T, K):
    x = activations(gen(T, K), T, K, torch.float32)
    q = ops.quantize_e4m3(x)
    zero = torch.zeros(T, K, dtype=torch.float64)
    assert coded_error(q, x.double(), zero) <= 0 and scale_error(q, x.double(), zero) <= 0
    assert torch.equal(q.values().double(), values64(q).float().double())
    assert q.codes.float().abs().amax() == 448


def test_rows_of_zeros_and_of_what_is_not_finite():
    x = torch.zeros(3, 130)
    x[1, 3], x[1, 129], x[2, 4], x[2, 5] = float("inf"), float("nan"), 1e-38, -1e-38
    q = ops.quantize_e4m3(x)
    assert torch.equal(q.codes[0].float(), torch.zeros(130)) and torch.isfinite(q.scale).all() and (q.scale > 0).all()
    assert torch.isnan(q.codes[1].float()).sum() == 2 and torch.equal(q.codes[2].float(), torch.zeros(130))


def test_norm_rounds_the_stream_once():
    g = gen(1)
    x, r, w = torch.randn(4, 256, generator=g).bfloat16(), torch.randn(4, 256, generator=g), torch.randn(256, generator=g)
    q, y, h = ops.rmsnorm_e4m3(x, w, 1e-6, r, want_rows=True)
    assert torch.equal(h, (x.float() + r).bfloat16())
    want = ops.rmsnorm(h.float(), w, 1e-6)
    assert torch.equal(y, want.bfloat16()) and torch.equal(q.codes.float(), ops.quantize_e4m3(want).codes.float())


def test_chain_of_a_layer():
    """norm, gated product and down product as they follow one another, each against 64 bits of what the one before left."""
    g = gen(2)
    x, gain = activations(g, 6, 256, torch.float32), 1 + 0.1 * torch.randn(256, generator=g)
    gu, dn = weight(g, 768, 256), weight(g, 256, 384)
    q = ops.rmsnorm_e4m3(x, gain, 1e-6)[0]
    h = ops.linear_gated_e4m3(q, gu)
    y, tol = sum_tol(q, gu)
    want = torch.nn.functional.silu(y[:, :384]) * y[:, 384:]
    err = 1.2 * tol[:, :384] * (y[:, 384:].abs() + tol[:, 384:]) + y[:, :384].abs() * tol[:, 384:] + 2.0 ** -20 * want.abs()
    assert coded_error(h, want, err) <= 0 and scale_error(h, want, err) <= 0
    out = ops.linear_e4m3(h, dn, residual=x, res_scale=0.5)
    want, tol = sum_tol(h, dn)
    want = want + 0.5 * x.double()
    assert bool(((out.double() - want).abs() <= tol + 2.0 ** -22 * (want.abs() + x.double().abs())).all())


def test_an_empty_share_of_the_columns_adds_nothing():
    """What a rank without features of a gated product, or without columns of a row-parallel one, has to do."""
    g = gen(4)
    q, r, b = rows(torch.randn(3, 128, generator=g)), torch.randn(3, 64, generator=g), torch.randn(64, generator=g)
    none = ops.linear_gated_e4m3(q, LinearWeight("fp8a", torch.zeros(0, 128).to(torch.float8_e4m3fn), torch.zeros(0, 1), in_features=128, out_features=0))
    assert none.shape == (3, 0) and none.scale.shape == (0, 3)
    W = LinearWeight("fp8a", torch.zeros(64, 0).to(torch.float8_e4m3fn), torch.zeros(1, 0), in_features=0, out_features=64)
    assert torch.equal(ops.linear_e4m3(none, W), torch.zeros(3, 64))
    assert torch.equal(ops.linear_e4m3(none, W, b, "relu", r, 0.5), b.clamp_min(0) + 0.5 * r)


def test_refusals():
    g = gen(3)
    q, W = rows(torch.randn(4, 256, generator=g)), weight(g, 512, 256)
    odd = weight(g, 320, 256)
    with pytest.raises(ValueError, match="codes"):
        ops.RowsE4M3(torch.zeros(4, 256), q.scale)
    for scale in (q.scale[:1], q.scale.double(), q.scale.t()):
        with pytest.raises(ValueError, match="scales"):
            ops.RowsE4M3(q.codes, scale)
    with pytest.raises(ValueError, match="rows in e4m3"):
        ops.linear_e4m3(torch.zeros(4, 256), W)
    with pytest.raises(ValueError, match="e4m3 with a scale"):
        ops.linear_e4m3(q, make_linear(torch.zeros(8, 256), "fp32"))
    with pytest.raises(ValueError, match="columns"):
        ops.linear_e4m3(q, weight(g, 512, 128))
    with pytest.raises(ValueError, match="activation"):
        ops.linear_e4m3(q, W, act="softcap")
    with pytest.raises(ValueError, match="bias"):
        ops.linear_e4m3(q, W, torch.zeros(511))
    with pytest.raises(ValueError, match="bias"):
        ops.linear_e4m3(q, W, torch.zeros(512).bfloat16())
    with pytest.raises(ValueError, match="residual"):
        ops.linear_e4m3(q, W, residual=torch.zeros(5, 512))
    with pytest.raises(ValueError, match="bf16 or fp32"):
        ops.linear_e4m3(q, W, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.linear_gated_e4m3(q, odd)
    with pytest.raises(ValueError, match="gain"):
        ops.rmsnorm_e4m3(torch.zeros(4, 256), torch.zeros(255), 1e-6)
    with pytest.raises(ValueError, match="residual"):
        ops.rmsnorm_e4m3(torch.zeros(4, 256), torch.zeros(256), 1e-6, torch.zeros(3, 256))
    with pytest.raises(ValueError, match="rows of"):
        ops.quantize_e4m3(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="end inside a block"):
        cat_linear([odd, W])
    for scale in (W.scale[:, :1], W.scale.double(), W.scale.t().contiguous().t(), W.scale[:1]):
        with pytest.raises(ValueError, match="scales"):
            ops.linear_e4m3(q, scaled(W, scale))
    for kw in (dict(times=torch.zeros(4, 512)), dict(out=torch.zeros(4, 512))):
        with pytest.raises(ValueError, match="no `out` and no `times`"):
            ops.linear(q, W, **kw)
    e = [(W, weight(g, 256, 256))]
    idx, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    for bad, match in ((dict(q=rows(torch.zeros(4, 128))), "columns"), (dict(idx=idx[:3]), "experts"), (dict(w=w[:, :1]), "weights"),
                       (dict(idx=idx[:, :0], w=w[:, :0]), "experts"), (dict(add=torch.zeros(4, 128)), "added"), (dict(experts=[]), "no experts"),
                       (dict(out_dtype=torch.float16), "bf16 or fp32"), (dict(act="clamped"), "activation"),
                       (dict(experts=[(odd, weight(g, 256, 160))]), "multiples of 128"),
                       (dict(experts=e + [(weight(g, 256, 256), weight(g, 256, 128))]), "different sizes"), (dict(packed={}), "packed"),
                       (dict(packed=dict(gus=None, E=2)), "packed"), (dict(experts=[(scaled(W, W.scale[:1, :1]), e[0][1])]), "scales")):
        with pytest.raises(ValueError, match=match):
            ops.moe_experts_e4m3(**{**dict(q=q, idx=idx, w=w, experts=e), **bad})


def test_mirror_of_the_kernels_parameters():
    from xfastertransformer_b200.ops import native as N
    from xfastertransformer_b200.ops.native_e4m3 import ROWS_ARGS, ROWS_GEMM
    fn = N.lib().xft_rows_gemm_layout
    got = (C.c_longlong * 64)()
    n = fn(got, 64)
    sizes = [8] * 12 + [8] * 2 + [4] * 18 + [4]                       # pointers, pitches, sizes, a factor: what ROWS_GEMM packs
    assert n == 1 + len(sizes) and ROWS_GEMM.format == "@12P2q18if"
    assert list(got[1:n]) == [sum(sizes[:i]) for i in range(len(sizes))]
    n = N.lib().xft_rows_args_layout(got, 64)
    rows = [8] * 13 + [4] * 4
    assert n == 1 + len(rows) and ROWS_ARGS.format == "@7P6q3if" and got[0] == ROWS_ARGS.size == sum(rows)
    assert list(got[1:n]) == [sum(rows[:i]) for i in range(len(rows))]
    n = fn(got, 64)
    assert ROWS_GEMM.size == sum(sizes) and ROWS_GEMM.size <= got[0] <= ROWS_GEMM.size + 4      # the struct may be padded at its end


# -- models -----------------------------------------------------------------------------------------------------------
def deepseek(layers=3, q_lora=256, **over):
    kw = dict(model_type="deepseek_moe", num_layer=layers, hidden_size=256, head_num=4, kv_head_num=4, size_per_head=128, inter_size=512,
              vocab_size=512, max_pos_seq_len=4096, q_lora_rank=q_lora, kv_lora_rank=128, qk_nope_head_dim=128, qk_rope_head_dim=64,
              v_head_dim=128, moe_intermediate_size=128, first_k_dense_replace=1, dense_experts=1, sparse_experts=8, routed_scaling_factor=2.5,
              topk_method="noaux_tc", n_group=4, topk_group=2, num_experts_per_tok=3, norm_topk_prob=True, scoring_func="sigmoid",
              activation_type="silu", weight_data_type="fp8_e4m3", start_id=0, end_id=1, rope=RopeConfig(theta=10000))
    return ModelConfig(**{**kw, **over})


def checkpoint(path, cfg, dtype):
    write_synthetic_checkpoint(str(path), cfg, seed=0, dtype=dtype, std=0.05)
    return str(path)


def logits(model, ids):
    """Prompt logits, and those of two steps."""
    sid = model.set_input_cb(ids, None, 64)
    out = [model.forward_cb().cpu().float()]
    for t in (7, 11):
        model.set_input_cb([[t]] * len(ids), sid, 64)
        out.append(model.forward_cb().cpu().float())
    model.free_seqs(sid)
    return out


IDS = [[5, 9, 300, 41, 77], [13, 8, 2, 450, 19, 33, 21]]


@pytest.mark.parametrize("family", ["llama", "llama-odd", "qwen2", "mixtral", "deepseek", "deepseek-direct", "opt"])
def test_model_is_its_operators(family, tmp_path, monkeypatch):
    """Norm, quantisation and product in few calls give what the single steps give (XFT_FUSE_NORM=0: norms and experts' sums on their own,
    activations quantised in front of each product).  DeepSeek: also what the type whose weights alone are e4m3 gives when its products see
    the values that rows in e4m3 stand for."""
    if family.startswith("deepseek"):
        cfg, dtype = deepseek(q_lora=256 if family == "deepseek" else 0), "fp8_e4m3"
    else:
        size = dict(num_layer=2, hidden_size=256, head_num=4, kv_head_num=2, size_per_head=64, inter_size=384, vocab_size=512, max_pos_seq_len=256)
        dtype = "bf16"
        cfg = {"llama": lambda: ModelConfig(model_type="llama", **size), "llama-odd": lambda: ModelConfig(model_type="llama", **{**size, "inter_size": 344}),
               "qwen2": lambda: ModelConfig(model_type="qwen2", **size),
               "mixtral": lambda: ModelConfig(model_type="mixtral", sparse_experts=4, num_experts_per_tok=2, **size),
               "opt": lambda: ModelConfig(model_type="gpt", **{**size, "kv_head_num": 4, "activation_type": "relu"})}[family]()
        cfg.weight_data_type = dtype
    d = checkpoint(tmp_path / "m", cfg, dtype)
    calls = []
    for name in ("rmsnorm_e4m3", "linear_e4m3", "linear_gated_e4m3", "moe_experts_e4m3"):
        fn = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, _f=fn, _n=name, **k: (calls.append(_n), _f(*a, **k))[1])
    got = logits(xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8"), IDS)
    used = set(calls)
    want_used = {"llama": {"rmsnorm_e4m3", "linear_e4m3", "linear_gated_e4m3"}, "llama-odd": {"rmsnorm_e4m3", "linear_e4m3"}, "opt": set()}
    assert used >= want_used.get(family, {"rmsnorm_e4m3", "linear_e4m3", "linear_gated_e4m3"} if family == "qwen2" else
                                 {"rmsnorm_e4m3", "linear_e4m3", "moe_experts_e4m3"})
    monkeypatch.setenv("XFT_FUSE_NORM", "0")
    Env._inst = None
    apart = logits(xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8"), IDS)
    for a, b in zip(got, apart):
        # the same values are quantised; sums that are taken in another order may move a value past the border of two codes
        assert (a - b).norm() <= 0.02 * b.norm()
    if dtype == "fp8_e4m3":
        for name in ("linear", "linear_gated"):
            fn = getattr(R, name)
            monkeypatch.setattr(R, name, lambda x, W, *a, _f=fn, **k: _f(R.quantize_e4m3(x).values() if W.kind == "fp8" else x, W, *a, **k))
        seen = logits(xft.AutoModel.from_pretrained(d, dtype="fp8_e4m3"), IDS)
        for a, b in zip(got, seen):
            assert (a - b).norm() <= 0.02 * b.norm()


def test_experts_output_waits_for_the_next_norm(tmp_path, monkeypatch):
    """The stream that a layer hands on lacks the experts' sum until the next norm adds it: the same logits as when each layer adds its own, and
    nothing is left behind by a pass that raised."""
    d = checkpoint(tmp_path / "m", deepseek(), "fp8_e4m3")
    m = xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8")
    got = logits(m, IDS)
    dec = m.model.decoder
    assert dec._pending is None
    monkeypatch.setenv("XFT_DEBUG_DIR", str(tmp_path / "dump"))          # dumps want the stream itself
    Env.get().reload()
    try:
        whole = logits(m, IDS)
    finally:
        monkeypatch.delenv("XFT_DEBUG_DIR")
        Env.get().reload()
    for a, b in zip(got, whole):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * b.abs().max().item())
    route, n = ops.route, []

    def third(*a, **k):
        n.append(1)
        if len(n) == 2:
            raise RuntimeError("lost")
        return route(*a, **k)

    monkeypatch.setattr(ops, "route", third)
    sid = m.set_input_cb(IDS, None, 64)
    with pytest.raises(RuntimeError, match="lost"):
        m.forward_cb()
    monkeypatch.setattr(ops, "route", route)
    m.free_seqs(sid)
    for a, b in zip(logits(m, IDS), got):
        assert torch.equal(a, b)


def test_types_that_have_no_such_form(tmp_path):
    d = checkpoint(tmp_path / "k", preset("tiny-kafipel"), "bf16")
    with pytest.raises(Exception, match="fp8_w8a8"):
        xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8")
