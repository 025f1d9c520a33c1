"""Models of dtype "fp8_w8a8" on a GPU: every call that a pass makes of the e4m3 operators against 64 bits of that call's own inputs, and captured
decode steps against eager ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import xfastertransformer_b200 as xft
from e4m3_rows import coded_error, dense64, scale_error, sum_tol, values64
from test_e4m3_rows_cpu import checkpoint, deepseek
from xfastertransformer_b200 import ops
from xfastertransformer_b200.config import ModelConfig
from xfastertransformer_b200.ops import reference as R
from xfastertransformer_b200.utils.flags import Env


def config(family):
    if family == "deepseek":
        return deepseek(hidden_size=512, head_num=8, kv_head_num=8, kv_lora_rank=512), "fp8_e4m3"
    size = dict(num_layer=2, hidden_size=512, head_num=4, kv_head_num=2, size_per_head=128, inter_size=640, vocab_size=512, max_pos_seq_len=1024,
                weight_data_type="bf16")
    if family == "mixtral":
        return ModelConfig(model_type="mixtral", sparse_experts=4, num_experts_per_tok=2, **size), "bf16"
    if family == "llama-odd":
        size["inter_size"] = 568
    return ModelConfig(model_type="llama", **size), "bf16"


def checked(monkeypatch, seen):
    """Wraps the operators so that each call is checked; bf16 results may be off by half a step of bf16 more."""
    def wrap(name, check):
        fn = getattr(ops, name)

        def call(*a, **k):
            r = fn(*a, **k)
            seen.append(name)
            check(r, *a, **k)
            return r

        monkeypatch.setattr(ops, name, call)

    def norm(r, x, w, eps, residual=None, want_rows=False):
        q, y, h = r
        stream = x if residual is None else h
        if residual is not None:
            assert torch.equal(h, (x.float() + residual.float()).bfloat16())
        d = stream.cpu().double()
        want = d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps) * w.cpu().double()
        err = (x.shape[-1] / 256 + 21) * 2.0 ** -24 * want.abs()
        assert coded_error(q, want, err) <= 0 and scale_error(q, want, err) <= 0

    def linear(r, q, W, bias=None, act=None, residual=None, res_scale=1.0, out_dtype=None):
        assert bias is None and act is None
        want, tol = sum_tol(q, W)
        if residual is not None:
            want = want + res_scale * residual.cpu().double()
            tol = tol + 2.0 ** -23 * (want.abs() + residual.cpu().double().abs())
        half = 0.0 if r.dtype == torch.float32 else 2.0 ** -8
        assert bool(((r.cpu().double() - want).abs() <= tol + half * want.abs()).all())

    def gated(r, q, W, act="silu", bias=None):
        y, tol = sum_tol(q, W)
        i = y.shape[1] // 2
        want = torch.nn.functional.silu(y[:, :i]) * y[:, i:]
        err = 1.2 * tol[:, :i] * (y[:, i:].abs() + tol[:, i:]) + y[:, :i].abs() * tol[:, i:] + 2.0 ** -18 * y[:, :i].abs() * y[:, i:].abs()
        assert coded_error(r, want, err) <= 0 and scale_error(r, want, err) <= 0

    def experts(r, q, idx, w, experts, act="silu", expert_offset=0, packed=None, expected_pairs=None, add=None, out_dtype=torch.float32):
        # the middle row may be off by its error and half a step of e4m3 (relative 2^-4, 2^-10 of a scale that is at most max / 448)
        out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        x, idx, w = values64(q), idx.cpu(), w.cpu().double()
        for e, (gu, dn) in enumerate(experts):
            tok, slot = (idx == e + expert_offset).nonzero(as_tuple=True)
            if not tok.numel():
                continue
            y = x[tok] @ dense64(gu).t()
            t = (136 + 3 * q.scale.shape[0]) * 2.0 ** -24 * (x[tok].abs() @ dense64(gu).abs().t())
            i = y.shape[1] // 2
            h = torch.nn.functional.silu(y[:, :i]) * y[:, i:]
            off = 1.2 * t[:, :i] * (y[:, i:].abs() + t[:, i:]) + y[:, :i].abs() * t[:, i:] + 2.0 ** -18 * y[:, :i].abs() * y[:, i:].abs()
            top = (h.abs() + off).view(h.shape[0], -1, 128).amax(-1).repeat_interleave(128, 1)
            off = off + torch.maximum(2.0 ** -4 * (h.abs() + off), 2.0 ** -10 * top / 448) * 1.01
            d, f = dense64(dn), w[tok, slot][:, None]
            out.index_add_(0, tok, (h @ d.t()) * f)
            tol.index_add_(0, tok, (off @ d.abs().t() + 2.0 ** -7 * (h @ d.t()).abs() + 2.0 ** -16 * (h.abs() @ d.abs().t())) * f)
        if add is not None:
            out = out + add.cpu().double()
        assert bool(((r.cpu().double() - out).abs() <= tol + 2.0 ** -20 * out.abs()).all())

    for name, check in (("rmsnorm_e4m3", norm), ("linear_e4m3", linear), ("linear_gated_e4m3", gated), ("moe_experts_e4m3", experts)):
        wrap(name, check)


def steps(m, ids, new):
    sid = m.set_input_cb(ids, None, 600)
    out = [m.forward_cb().cpu()]
    for t in new:
        m.set_input_cb([[t + i] for i in range(len(ids))], sid, 600)
        out.append(m.forward_cb().cpu())
    m.free_seqs(sid)
    return out


def prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("family", ["llama", "llama-odd", "mixtral", "deepseek"])
def test_every_call_of_a_pass(family, tmp_path, monkeypatch):
    cfg, dtype = config(family)
    d = checkpoint(tmp_path / "m", cfg, dtype)
    monkeypatch.setenv("XFT_CUDA_GRAPH", "0")
    Env._inst = None
    m = xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8", kv_cache_dtype="bf16")
    plain = steps(m, prompts(150, 41, 7), (3, 90))
    seen = []
    checked(monkeypatch, seen)
    again = steps(m, prompts(150, 41, 7), (3, 90))
    want = {"rmsnorm_e4m3", "linear_e4m3"} | ({"linear_gated_e4m3"} if family in ("llama", "deepseek") else set()) | \
        ({"moe_experts_e4m3"} if family in ("mixtral", "deepseek") else set())
    assert set(seen) == want
    for a, b in zip(plain, again):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    from xfastertransformer_b200.ops import native as N
    N.Workspace.get(torch.device("cuda", 0)).check_status()


@pytest.mark.parametrize("family", ["llama", "mixtral", "deepseek"])
def test_captured_steps_are_the_eager_ones(family, tmp_path, monkeypatch):
    cfg, dtype = config(family)
    d = checkpoint(tmp_path / "m", cfg, dtype)
    got = steps(xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8", kv_cache_dtype="bf16"), prompts(20, 33), range(3, 60, 7))
    ids = torch.tensor(prompts(24, 24))
    m = xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8", kv_cache_dtype="bf16")
    text = m.generate(ids, max_length=40)
    assert text.shape == (2, 40)
    monkeypatch.setenv("XFT_CUDA_GRAPH", "0")
    Env._inst = None
    eager = steps(xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8", kv_cache_dtype="bf16"), prompts(20, 33), range(3, 60, 7))
    for a, b in zip(got, eager):
        assert torch.equal(a, b)
