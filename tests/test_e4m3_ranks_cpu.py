"""Models of dtype "fp8_w8a8" on two gloo ranks against one rank on the same files: shares of the features in blocks of 128 (some of them empty), experts
that are sliced or whole, rows that travel to their experts, prompts whose sums overlap, and stages; and the shares themselves."""
import os
import subprocess
import sys

import pytest
import torch

import xfastertransformer_b200 as xft
from e4m3_rows import gen, rows, weight
from test_e4m3_rows_cpu import checkpoint, deepseek
from xfastertransformer_b200 import ops
from xfastertransformer_b200.config import ModelConfig
from xfastertransformer_b200.models.decoder import Decoder
from xfastertransformer_b200.parallel import partition as P
from xfastertransformer_b200.parallel.dist import DistContext
from xfastertransformer_b200.runtime.loader import LinearWeight
from xfastertransformer_b200.utils.flags import Env

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("n", [128, 256, 384, 2048, 8192, 11008, 14336, 18432, 28672])
@pytest.mark.parametrize("ranks", [1, 2, 4, 8])
def test_shares_of_blocks(n, ranks):
    """They follow one another, cover everything, differ by a block at most, and are empty only where there are fewer blocks than ranks."""
    parts = [P.block_range(n, 128, ranks, i) for i in range(ranks)]
    assert parts[0][0] == 0 and parts[-1][1] == n and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
    sizes = [(e - s) // 128 for s, e in parts]
    assert all((e - s) % 128 == 0 for s, e in parts) and max(sizes) - min(sizes) <= 1 and (min(sizes) > 0) == (n // 128 >= ranks)
    dec = Decoder.__new__(Decoder)
    dec.kind, dec.tp = "fp8a", ranks
    for i in range(ranks):
        dec.tpr = i
        assert dec._ffn_range(n, 128) == parts[i]
        dec.kind = "fp8"                                               # weights alone in e4m3: where the reference would cut
        assert dec._ffn_range(n, 128) == P.task_range_gran(n, 128, ranks, i)
        dec.kind = "fp8a"


def test_refusals_of_shares():
    for bad in ((100, 128, 2, 0), (256, 128, 0, 0), (256, 128, 2, 2), (256, 128, 2, -1)):
        with pytest.raises(ValueError):
            P.block_range(*bad)


def test_a_product_of_an_empty_share_counts_its_rows(monkeypatch, capsys):
    """The sum over the ranks and the printed line ask for the rows of a share without columns."""
    none = ops.linear_gated_e4m3(rows(torch.randn(3, 128, generator=gen(1))),
                                 LinearWeight("fp8a", torch.zeros(0, 128).to(torch.float8_e4m3fn), torch.zeros(0, 1), in_features=128, out_features=0))
    no_columns = lambda n: LinearWeight("fp8a", torch.zeros(n, 0).to(torch.float8_e4m3fn), torch.zeros(-(-n // 128), 0), in_features=0, out_features=n)
    W = no_columns(64)

    class Peer:
        slot = 0
        asked = []

        def can_fuse(self, T, n, kind):
            self.asked.append((T, n, kind))
            return False

        def can_fuse_bulk(self, T, n, k, kind):
            self.asked.append((T, n, k, kind))
            return False

    class Rows:                                                        # as rows on a GPU are seen
        is_cuda, shape = True, none.shape

        def numel(self):
            return 0

    dec = Decoder.__new__(Decoder)
    dec.tp, dec.tpr, dec._overlap = 2, 1, False
    dec.ctx = type("Ctx", (), dict(peer=Peer(), all_reduce=staticmethod(lambda y: y)))()
    linear = ops.linear
    monkeypatch.setattr(ops, "linear", lambda h, *a, **k: linear(none if isinstance(h, Rows) else h, *a, **k))
    assert torch.equal(dec._row_parallel(Rows(), W, None, None), torch.zeros(3, 64))
    assert Peer.asked == [(3, 64, "fp8a"), (3, 64, 0, "fp8a")]
    monkeypatch.setattr(ops, "linear", linear)
    monkeypatch.setenv("XFT_VERBOSE", "1")
    Env.get().reload()
    try:
        assert torch.equal(ops.linear_gated_e4m3(none, no_columns(256)).codes.float(), torch.zeros(3, 128))
    finally:
        monkeypatch.delenv("XFT_VERBOSE")
        Env.get().reload()
    assert "m3n256k0" in "".join(capsys.readouterr())


def config(family):
    # heads of 128: each rank's queries, keys and values are whole blocks of weights, which are quantised alike on one rank and on two
    size = dict(num_layer=2, hidden_size=512, head_num=4, kv_head_num=2, size_per_head=128, inter_size=384, vocab_size=512, max_pos_seq_len=256,
                weight_data_type="bf16", start_id=0, end_id=1)
    if family == "deepseek":
        return deepseek(), "fp8_e4m3"
    if family.startswith("mixtral"):
        return ModelConfig(model_type="mixtral", sparse_experts=4, num_experts_per_tok=2, **{**size, "inter_size": 128 if family == "mixtral-thin" else 384}), "bf16"
    return ModelConfig(model_type="llama", **{**size, "inter_size": {"llama-thin": 128, "llama-odd": 344}.get(family, 384)}), "bf16"


CASES = [("llama", "tp"), ("llama-thin", "tp"), ("llama-odd", "tp"), ("llama", "overlap"), ("mixtral", "tp"), ("mixtral-thin", "tp"), ("mixtral-thin", "apart"),
         ("deepseek", "tp"), ("deepseek", "ep"), ("deepseek", "dp"), ("mixtral", "dp"), ("deepseek", "overlap"), ("deepseek", "pp"), ("deepseek", "apart")]


@pytest.mark.parametrize("family,mode", CASES)
def test_two_ranks_are_one(family, mode, tmp_path, monkeypatch):
    """The ranks quantise the same values in the same blocks, so their sums differ by the order of addition alone, which may move a value past the
    border of two codes; "apart": norms and experts' sums on their own (XFT_FUSE_NORM=0)."""
    cfg, dtype = config(family)
    d, out = checkpoint(tmp_path / "m", cfg, dtype), str(tmp_path / "out.pt")
    env = dict(os.environ, XFT_ENGINE="CPU", XFT_EXPERT_PARALLEL=str(int(mode == "ep")), XFT_ATTENTION_DP=str(int(mode == "dp")),
               XFT_PREFILL_OVERLAP=str(int(mode == "overlap")), XFT_PIPELINE_STAGE="2" if mode == "pp" else "1",
               XFT_FUSE_NORM=str(int(mode != "apart")), OMP_NUM_THREADS="2", PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port",
           str(29761 + CASES.index((family, mode))), os.path.join(ROOT, "tests", "e4m3_ranks_worker.py"), d, out]
    r = subprocess.run(cmd, env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    got = torch.load(out)
    monkeypatch.setenv("XFT_ENGINE", "CPU")
    DistContext.reset()
    m = xft.AutoModel.from_pretrained(d, dtype="fp8_w8a8")
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (21, 5, 13)]
    sid = m.set_input_cb(prompts, None, 64)
    want = [m.forward_cb().float()]
    for t in (7, 11):
        m.set_input_cb([[t], [t + 1], [t + 2]], sid, 64)
        want.append(m.forward_cb().float())
    m.free_seqs(sid)
    for a, b in zip(got["logits"], want):
        assert torch.isfinite(a).all()
        if family != "llama-odd":                                      # whose shares end inside a block: other weights share a scale
            assert (a - b).norm() <= 0.02 * b.norm()
    assert got["tokens"].shape == (2, 10)
    held = got["held"]
    assert not any(h["left"] for h in held)
    sliced = mode in ("tp", "overlap", "apart")
    if family == "llama" or family == "llama-thin":
        assert [h["down"] for h in held] == ([[256, 256], [128, 128]] if family == "llama" else [[128, 128], [0, 0]])
    if family == "llama-odd":
        assert [h["down"] for h in held] == [[172, 172], [172, 172]]
    if family == "mixtral-thin":                                       # whose turn it is goes round with the layer
        assert [h["experts"] for h in held] == [(0, 4, [128] * 4), (0, 4, [0] * 4)]
    if family == "deepseek" and sliced:
        assert [h["down"][0] for h in held] == [256, 256] and sorted(h["shared"] for h in held) == [0, 128]
        assert sorted(h["experts"][2][0] for h in held) == [0, 128]
    if mode in ("ep", "dp"):
        n = cfg.sparse_experts // 2
        assert [h["experts"][:2] for h in held] == [(0, n), (n, n)] and all(w == held[0]["experts"][2][0] for h in held for w in h["experts"][2])
    assert all((h["sent"] > 0) == (mode == "dp") for h in held) and all((h["pairs"] > 0) == (mode == "overlap") for h in held)
    if mode == "pp":
        assert held[0]["layers"][1] == held[1]["layers"][0] > 0
