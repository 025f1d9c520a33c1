"""Rows in e4m3 and their products on a GPU (csrc/kernels/rows_e4m3.cu, gemm_e4m3_sm100.cu, gemm_rows_e4m3_sm100.cu) against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import activations, coded_error, dense64, gen, on, rows, rows_on, scale_error, sum_tol, values64, weight
from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import reference as R
from xfastertransformer_b200.runtime.loader import LinearWeight, make_linear


def check_status():
    from xfastertransformer_b200.ops import native as N
    N.Workspace.get(torch.device("cuda", 0)).check_status()


# every number of threads and columns per thread, a block cut short, one column of eight
@pytest.mark.parametrize("T,K", [(1, 8), (3, 128), (2, 200), (5, 504), (4, 1032), (7, 2112), (3, 4104), (300, 896), (2, 8200), (2, 16392), (1, 32768)])
def test_codes_are_the_formulas(T, K):
    """Without a norm nothing rounds but the formula's own steps, which IEEE arithmetic fixes: the same bits as on a CPU."""
    x = activations(gen(T, K), T, K)
    got, want = ops.quantize_e4m3(x.cuda()), ops.quantize_e4m3(x)
    assert torch.equal(got.codes.cpu().view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scale.cpu(), want.scale)


def test_codes_of_extreme_rows():
    """Zeros, values below the floor, the largest bf16, and values that are not finite, which become NaN and leave the others alone."""
    x = torch.zeros(6, 264).bfloat16()
    x[1] = 1e-38
    x[2] = torch.finfo(torch.bfloat16).max
    x[3, ::2], x[3, 1::2] = -3.0, 0.001
    x[4] = torch.randn(264, generator=gen(4)).bfloat16()
    x[4, 5], x[4, 130], x[4, 263] = float("inf"), float("nan"), float("-inf")
    x[5, 200] = float("nan")
    got, want = ops.quantize_e4m3(x.cuda()), ops.quantize_e4m3(x)
    c, w = got.codes.cpu().float(), want.codes.float()
    assert torch.equal(torch.isnan(c), torch.isnan(w)) and torch.equal(torch.nan_to_num(c), torch.nan_to_num(w))
    assert torch.equal(got.scale.cpu(), want.scale)
    assert torch.isnan(c[4]).sum() == 3 and torch.isnan(c[5]).sum() == 1 and torch.isfinite(got.scale).all()


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 128), (2, 8), (33, 1000), (5, 4096), (130, 7168), (2, 16384)])
def test_norm_matches_64_bits(T, K, residual):
    """The fp32 norm is off by a few roundings and by those of its sum, at most K / 256 additions in a row of threads and 13 joins."""
    g = gen(T, K, 0 if residual is None else 1)
    x = activations(g, T, K)
    if T > 3:
        x[2] = torch.randn(K, generator=g).bfloat16()              # squares of 1e20 leave 32 bits
    gain = (1 + 0.2 * torch.randn(K, generator=g))
    r = None if residual is None else (torch.randn(T, K, generator=g) * x.float().abs().mean()).to(residual)
    q, y, h = ops.rmsnorm_e4m3(x.cuda(), gain.cuda(), 1e-6, None if r is None else r.cuda(), want_rows=True)
    stream = x if r is None else (x.double() + r.double()).float().bfloat16()
    if r is None:
        assert h is None
    else:
        assert torch.equal(h.cpu(), (x.float() + r.float()).bfloat16())
        stream = h.cpu()
    d = stream.double()
    want = d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + 1e-6) * gain.double()
    err = (K / 256 + 13 + 8) * 2.0 ** -24 * want.abs()
    assert coded_error(q, want, err) <= 0 and scale_error(q, want, err) <= 0
    assert bool(((y.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + err).all())
    again = ops.rmsnorm_e4m3(x.cuda(), gain.cuda(), 1e-6, None if r is None else r.cuda())
    assert again[1] is None and torch.equal(again[0].codes.view(torch.uint8), q.codes.view(torch.uint8))


def test_norm_of_strided_rows():
    """Slices of wider rows, at and between 16 bytes, as the projections leave them: the bits of a copy."""
    g = gen(9)
    wide, gain = activations(g, 20, 1200).cuda(), torch.randn(520, generator=g).cuda()
    res = torch.randn(20, 1200, generator=g).cuda()
    for at in (0, 8, 3):
        x, r = wide[:, at:at + 520], res[:, at:at + 520]
        a, b = ops.rmsnorm_e4m3(x, gain, 1e-5, r), ops.rmsnorm_e4m3(x.clone(), gain, 1e-5, r.clone())
        assert torch.equal(a[0].codes.view(torch.uint8), b[0].codes.view(torch.uint8)) and torch.equal(a[0].scale, b[0].scale)
        assert torch.equal(a[2], b[2])
    off = torch.randn(521, generator=g).cuda()[1:]                 # a gain that starts between 16 bytes
    a, b = ops.rmsnorm_e4m3(wide[:, :520], off, 1e-5), ops.rmsnorm_e4m3(wide[:, :520], off.clone(), 1e-5)
    assert torch.equal(a[0].codes.view(torch.uint8), b[0].codes.view(torch.uint8))


# token tiles and one past them, features and k that end inside a block, k that wants a pitch of its own, few and many tiles, parts of k
SHAPES = [(1, 128, 128), (1, 2112, 4096), (16, 136, 8), (17, 384, 200), (32, 1000, 1032), (33, 200, 4096), (64, 264, 2056), (65, 512, 1152),
          (129, 136, 640), (200, 4096, 520), (257, 300, 1024), (300, 2112, 7168), (1000, 1544, 264), (2100, 640, 512), (150, 901, 1000), (333, 2049, 256),
          (2000, 1283, 136), (1, 33, 72)]


@pytest.mark.parametrize("T,N,K", SHAPES)
def test_product_matches_64_bits(T, N, K):
    g = gen(T, N, K)
    q, W = rows(activations(g, T, K)), weight(g, N, K)
    bias, res = torch.randn(N, generator=g), torch.randn(T, N, generator=g).bfloat16()
    want, tol = sum_tol(q, W)
    dq, dW = rows_on(q), on(W)
    got = ops.linear_e4m3(dq, dW, out_dtype=torch.float32)
    check_status()
    assert bool(((got.cpu().double() - want).abs() <= tol).all()), ((got.cpu().double() - want).abs() / tol).max().item()
    full = want + bias.double() + 0.5 * res.double()
    tol = tol + 2.0 ** -23 * (bias.double().abs() + res.double().abs() + want.abs())
    for dtype, half in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        got = ops.linear_e4m3(dq, dW, bias.cuda(), None, res.cuda(), 0.5, out_dtype=dtype)
        assert got.dtype == dtype and bool(((got.cpu().double() - full).abs() <= tol + half * full.abs()).all())
    check_status()


# tiles of prompts, whatever the size would choose: one item and several per CTA, rows and features that end inside a tile, one block of k and
# many, k that ends inside a block
@pytest.mark.parametrize("form", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("T,N,K", [(1, 8, 128), (100, 136, 16), (65, 200, 520), (131, 256, 3000), (129, 256, 640), (257, 300, 1032), (300, 2112, 2048), (2000, 5000, 264), (9000, 1160, 128), (140, 777, 1024),
                                   (513, 515, 640)])
def test_tiles_of_prompts(T, N, K, form):
    from xfastertransformer_b200.ops import native_e4m3 as E
    g = gen(T, N, K)
    q, W = rows(activations(g, T, K)), weight(g, N, K)
    bias, res = torch.randn(N, generator=g), torch.randn(T, N, generator=g).bfloat16()
    if form > 4 and -(-K // 128) < 2 * form - 8:
        pytest.skip("fewer blocks of k than parts")
    want, tol = sum_tol(q, W)
    want = want + bias.double() + 0.5 * res.double()
    tol = tol + 2.0 ** -23 * (bias.double().abs() + res.double().abs() + want.abs())
    dq, dW = rows_on(q), on(W)
    for dtype, half in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.full((T + 1, N), 7.0, dtype=dtype, device="cuda")
        E._gemm(dq, dW.w if K % 16 == 0 else E._weight(dW), dW.scale, out[:T], T, N, K, bias=bias.cuda(), residual=res.cuda(), res_scale=0.5, form=form)
        check_status()
        assert bool(((out[:T].cpu().double() - want).abs() <= tol + half * want.abs()).all()) and bool((out[T] == 7).all())


# rows of the result and of the residual that start anywhere between 16 bytes, each at its own place
@pytest.mark.parametrize("form", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("N,pitch,off", [(641, 647, 1), (642, 645, 3), (516, 520, 4), (768, 769, 0), (513, 520, 8), (70, 77, 5), (135, 135, 0)])
def test_rows_between_16_bytes(N, pitch, off, form):
    from xfastertransformer_b200.ops import native_e4m3 as E
    T, K = 261, 1024
    g = gen(N, pitch, off)
    q, W, bias = rows(activations(g, T, K)), weight(g, N, K), torch.randn(N, generator=g)
    wide = torch.randn(T, pitch + 8, generator=g).bfloat16()
    want, tol = sum_tol(q, W)
    want = (want + bias.double()).clamp_min(0) + 0.5 * wide[:, off:off + N].double()
    tol = tol + 2.0 ** -23 * (bias.double().abs() + wide[:, off:off + N].double().abs() + want.abs())
    dq, dW, dres = rows_on(q), on(W), wide.cuda()[:, off:off + N]
    for dtype, half in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        room = torch.full((T + 1, pitch), 7.0, dtype=dtype, device="cuda")
        out = room.view(-1)[1:1 + T * pitch].view(T, pitch)[:, :N]
        E._gemm(dq, dW.w, dW.scale, out, T, N, K, bias=bias.cuda(), act="relu", residual=dres, res_scale=0.5, form=form)
        check_status()
        assert bool(((out.cpu().double() - want).abs() <= tol + half * want.abs()).all())
        out.fill_(7)
        assert bool((room == 7).all())


@pytest.mark.parametrize("form", [1, 3])
@pytest.mark.parametrize("T,I,K", [(1, 128, 128), (130, 384, 200), (300, 640, 1024), (5000, 1408, 256)])
def test_gated_tiles_of_prompts(T, I, K, form):
    from xfastertransformer_b200.ops import native_e4m3 as E
    g = gen(T, I, K)
    q, W, bias = rows(torch.randn(T, K, generator=g)), weight(g, 2 * I, K), torch.randn(2 * I, generator=g)
    y, tol = sum_tol(q, W)
    y, tol = y + bias.double(), tol + 2.0 ** -23 * (y.abs() + bias.double().abs())
    a = R._act(y[:, :I], "silu")
    want = a * y[:, I:]
    err = 1.2 * tol[:, :I] * (y[:, I:].abs() + tol[:, I:]) + a.abs() * tol[:, I:] + 2.0 ** -18 * y[:, :I].abs() * y[:, I:].abs()
    dq, dW = rows_on(q), on(W)
    out = E.new_rows(T, I, dq.codes)
    E._gemm(dq, E._weight(dW), dW.scale, out.codes, T, I, K, True, I, bias.cuda(), "silu", out_scale=out.scale, form=form)
    check_status()
    assert coded_error(out, want, err) <= 0 and scale_error(out, want, err) <= 0
    plain = torch.empty(T, I, dtype=torch.bfloat16, device="cuda")
    E._gemm(dq, E._weight(dW), dW.scale, plain, T, I, K, True, I, bias.cuda(), "silu", form=form)
    check_status()
    assert bool(((plain.cpu().double() - want).abs() <= err + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("T", [5, 40, 150])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "relu2", "gelu_erf", "tanh"])
def test_activations(T, act):
    """|act'| is at most 1.2, but for relu2, 2 |y|; the functions themselves are good to 2^-18 of their largest part (|y|, or its square)."""
    g = gen(T, len(act))
    q, W = rows(torch.randn(T, 256, generator=g)), weight(g, 264, 256)
    y, tol = sum_tol(q, W)
    want = R._act(y, act)
    slope = 2 * y.abs() + tol if act == "relu2" else 1.2
    got = ops.linear_e4m3(rows_on(q), on(W), act=act, out_dtype=torch.float32).cpu().double()
    assert bool(((got - want).abs() <= slope * tol + 2.0 ** -18 * torch.maximum(y.abs(), y * y) + 2.0 ** -20).all())
    check_status()


def gated64(q, W, act):
    """(act(g) u in 64 bits, how far off it may be)"""
    y, tol = sum_tol(q, W)
    i = W.out_features // 2
    (gt, up), (tg, tu) = (y[:, :i], y[:, i:]), (tol[:, :i], tol[:, i:])
    a = R._act(gt, act)
    return a * up, 1.2 * tg * (up.abs() + tu) + a.abs() * tu + 2.0 ** -18 * torch.maximum(gt.abs(), a.abs()) * up.abs()


@pytest.mark.parametrize("T,I,K", [(1, 128, 128), (3, 128, 256), (16, 640, 4096), (31, 384, 4112), (64, 256, 1040), (65, 128, 200), (130, 640, 528), (257, 1408, 512), (700, 1024, 1024)])
def test_gated_matches_64_bits(T, I, K):
    g = gen(T, I, K)
    q, W = rows(activations(g, T, K) if T < 100 else torch.randn(T, K, generator=g)), weight(g, 2 * I, K)
    want, err = gated64(q, W, "silu")
    fine = want.abs().amax(1) < 1e30                                   # rows of 1e20 meet the end of 32 bits in their square
    got = ops.linear_gated_e4m3(rows_on(q), on(W), "silu")
    check_status()
    got = ops.RowsE4M3(got.codes.cpu()[fine], got.scale.cpu()[:, fine])
    assert fine.sum() >= T - 1
    assert coded_error(got, want[fine], err[fine]) <= 0 and scale_error(got, want[fine], err[fine]) <= 0


@pytest.mark.parametrize("T", [20, 70, 300])
def test_gated_bias_and_activation(T):
    g = gen(T)
    q, W, bias = rows(torch.randn(T, 256, generator=g)), weight(g, 512, 256), torch.randn(512, generator=g)
    y, tol = sum_tol(q, W)
    y = y + bias.double()
    want = R._act(y[:, :256], "relu") * y[:, 256:]
    tol = tol + 2.0 ** -23 * y.abs() + 2.0 ** -23 * bias.double().abs()
    err = tol[:, :256] * (y[:, 256:].abs() + tol[:, 256:]) + y[:, :256].abs() * tol[:, 256:] + 2.0 ** -23 * want.abs()
    got = ops.linear_gated_e4m3(rows_on(q), on(W), "relu", bias.cuda())
    check_status()
    assert coded_error(got, want, err) <= 0 and scale_error(got, want, err) <= 0


def whole(g, N, K, lo=-4, hi=4):
    """Weights whose codes and scales are small whole numbers and powers of two: sums of them are exact in fp32, in any order."""
    w = torch.randint(lo, hi + 1, (N, K), generator=g).float()
    s = 2.0 ** torch.randint(-3, 2, (-(-N // 128), -(-K // 128)), generator=g).float()
    return make_linear(w.to(torch.float8_e4m3fn), "fp8a", scale=s)


def whole_rows(g, T, K):
    c = torch.randint(-4, 5, (T, K), generator=g).float().to(torch.float8_e4m3fn)
    return ops.RowsE4M3(c, 2.0 ** torch.randint(-2, 3, (-(-K // 128), T), generator=g).float())


def routing(g, T, E, k, idle=True):
    """k of E experts per token, the last one asked by nobody, weights that do not add up to one."""
    score = torch.rand(T, E - 1 if idle and E - 1 >= k else E, generator=g)
    return score.topk(k, 1)[1].int(), torch.rand(T, k, generator=g) + 0.1


def experts64(q, idx, w, experts, offset=0):
    """Sum of the experts of whole-numbered inputs with relu, where the middle rows are exact before they are quantised, so that their codes are
    the formula's; and what the fp32 sums behind them may be off."""
    T = q.shape[0]
    H = experts[0][1].out_features
    out, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for e, (gu, dn) in enumerate(experts):
        tok, slot = (idx == e + offset).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        y = values64(q)[tok] @ dense64(gu).t()
        i = y.shape[1] // 2
        h = R.quantize_e4m3((y[:, :i].clamp_min(0) * y[:, i:]).float())
        s, t = sum_tol(h, dn)
        f = w[tok, slot].double()[:, None]
        out.index_add_(0, tok, s * f)
        tol.index_add_(0, tok, (t + 4 * 2.0 ** -24 * s.abs()) * f)
    return out, tol


# rows per expert on both sides of every tile: 16, 32, 64 and the tiles of prompts; sizes of one block, several, and of an odd number of blocks
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 128, 128), (3, 4, 1, 256, 384), (40, 8, 3, 384, 256), (90, 4, 2, 256, 128), (300, 4, 3, 640, 384),
                                       (700, 3, 2, 256, 640), (1500, 2, 1, 384, 256)])
def test_experts_match_64_bits(T, E, k, H, I):
    g = gen(T, E, k, H, I)
    q = whole_rows(g, T, H)
    experts = [(whole(g, 2 * I, H), whole(g, H, I)) for _ in range(E)]
    idx, w = routing(g, T, E, k)
    want, tol = experts64(q, idx, w, experts)
    dev = [(on(a), on(b)) for a, b in experts]
    got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), dev, "relu")
    check_status()
    big = tol + (k + 2) * 2.0 ** -24 * want.abs().amax(1, keepdim=True)
    half = experts_half_step(q, idx, w, experts)                    # prompts hold a pair's row in bf16 on its way into the sum
    assert bool(((got.cpu().double() - want).abs() <= big + half).all())
    add = torch.randn(T, H, generator=g)
    for a in (add, add.bfloat16()):
        for dtype, step in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
            full = want + a.double()
            got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), dev, "relu", add=a.cuda(), out_dtype=dtype)
            assert got.dtype == dtype
            assert bool(((got.cpu().double() - full).abs() <= (big + half + 2.0 ** -23 * full.abs()) * (1 + step) + step * full.abs()).all())
    check_status()


def experts_half_step(q, idx, w, experts, offset=0):
    """2^-8 of every pair's part of the sum."""
    T, H = q.shape[0], experts[0][1].out_features
    out = torch.zeros(T, H, dtype=torch.float64)
    for e, (gu, dn) in enumerate(experts):
        tok, slot = (idx == e + offset).nonzero(as_tuple=True)
        if tok.numel():
            y = values64(q)[tok] @ dense64(gu).t()
            i = y.shape[1] // 2
            h = R.quantize_e4m3((y[:, :i].clamp_min(0) * y[:, i:]).float())
            out.index_add_(0, tok, 2.0 ** -8 * (values64(h) @ dense64(dn).t()).abs() * w[tok, slot].double()[:, None])
    return out


@pytest.mark.parametrize("T", [6, 200])
def test_experts_of_a_part(T):
    """A rank's share of the experts: indexes outside it and -1 add nothing, tokens without a local expert get zeros, one expert twice counts twice."""
    g = gen(T)
    H, I, E = 256, 128, 3
    q, experts = whole_rows(g, T, H), [(whole(g, 2 * I, H), whole(g, H, I)) for _ in range(E)]
    idx, w = torch.randint(0, 9, (T, 3), generator=g).int(), torch.rand(T, 3, generator=g)
    idx[0], idx[1], idx[2] = 0, -1, 4
    want, tol = experts64(q, idx, w, experts, offset=3)
    got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), [(on(a), on(b)) for a, b in experts], "relu", expert_offset=3)
    check_status()
    assert torch.equal(got[0].cpu(), torch.zeros(H)) and torch.equal(got[1].cpu(), torch.zeros(H))
    bound = tol + 8 * 2.0 ** -24 * want.abs().amax(1, keepdim=True) + experts_half_step(q, idx, w, experts, 3)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


# one CTA and a cluster of them, one round of pairs and several, an expert and 256, tiles of every size, indexes on both sides of the local ones
@pytest.mark.parametrize("T,k,E,bn", [(1, 1, 1, 16), (5, 3, 4, 16), (31, 8, 256, 32), (1024, 2, 8, 64), (1025, 2, 8, 64), (2049, 1, 3, 128), (4096, 6, 64, 128),
                                      (9000, 8, 32, 256), (40000, 2, 2, 256)])
def test_plan_of_rows(T, k, E, bn):
    from xfastertransformer_b200.ops import native_e4m3 as E4
    g = gen(T, k, E)
    e0, n = 5, T * k
    idx = torch.randint(3, E + 7, (T, k), generator=g).int()
    idx[torch.rand(T, k, generator=g) < 0.1] = -1
    w = torch.rand(T, k, generator=g)
    most = (n + bn - 1) // bn + E
    i32 = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")
    pos, src, tiles, meta, row_w = i32(n), i32(n), i32(most, 4), i32(2), torch.full((n,), -7.0, device="cuda")
    di, dw = idx.cuda(), w.cuda()
    assert E4._lib().xft_plan_rows(di.data_ptr(), dw.data_ptr(), T, k, e0, e0 + E, bn, pos.data_ptr(), src.data_ptr(), row_w.data_ptr(), tiles.data_ptr(),
                                   meta.data_ptr(), most, E4._stream()) == 0
    pos, src, row_w, tiles, meta = (t.cpu() for t in (pos, src, row_w, tiles, meta))
    flat = idx.view(-1)
    local = (flat >= e0) & (flat < e0 + E)
    rows_ = int(local.sum())
    counts = torch.bincount((flat[local] - e0).long(), minlength=E)
    assert meta.tolist() == [int(((counts + bn - 1) // bn).sum()), rows_]
    assert bool((pos[~local] == -1).all()) and torch.equal(pos[local].sort()[0], torch.arange(rows_, dtype=torch.int32))
    start = torch.cumsum(counts, 0) - counts
    e = (flat[local] - e0).long()
    assert bool((pos[local] >= start[e]).all()) and bool((pos[local] < start[e] + counts[e]).all())
    pair = local.nonzero()[:, 0]
    at = pos[local].long()
    assert torch.equal(src[at], (pair // k).int()) and torch.equal(row_w[at], w.view(-1)[pair])
    want = [[i, int(start[i]) + j, min(bn, int(counts[i]) - j), 0] for i in range(E) for j in range(0, int(counts[i]), bn)]
    assert tiles[:len(want)].tolist() == want and bool((src[rows_:] == -7).all())


def test_experts_that_nobody_asks():
    g = gen(1)
    experts = [(on(whole(g, 256, 128)), on(whole(g, 128, 128))) for _ in range(2)]
    idx = torch.full((5, 2), 7, dtype=torch.int32, device="cuda")
    got = ops.moe_experts_e4m3(rows_on(whole_rows(g, 5, 128)), idx, torch.ones(5, 2, device="cuda"), experts)
    assert torch.equal(got.cpu(), torch.zeros(5, 128))
    check_status()


def test_no_rows():
    g = gen(2)
    W, q = on(weight(g, 256, 128)), ops.quantize_e4m3(torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 128) and ops.linear_e4m3(q, W).shape == (0, 256) and ops.linear_gated_e4m3(q, W).shape == (0, 128)
    n = ops.rmsnorm_e4m3(torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda"), torch.ones(128, device="cuda"), 1e-6,
                         torch.zeros(0, 128, device="cuda"), want_rows=True)
    assert n[0].shape == (0, 128) and n[1].shape == n[2].shape == (0, 128)
    e = [(W, on(weight(g, 128, 128)))]
    assert ops.moe_experts_e4m3(q, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), torch.zeros(0, 1, device="cuda"), e).shape == (0, 128)


def test_an_empty_share_of_the_columns_adds_nothing():
    g = gen(4)
    q = rows_on(whole_rows(g, 3, 128))
    none = ops.linear_gated_e4m3(q, LinearWeight("fp8a", torch.zeros(0, 128).to(torch.float8_e4m3fn), torch.zeros(0, 1), in_features=128,
                                                 out_features=0).to("cuda"))
    assert none.shape == (3, 0) and none.scale.shape == (0, 3)
    W = LinearWeight("fp8a", torch.zeros(64, 0).to(torch.float8_e4m3fn), torch.zeros(1, 0), in_features=0, out_features=64).to("cuda")
    r, b = torch.randn(3, 64, generator=g).bfloat16(), torch.randn(64, generator=g)
    assert torch.equal(ops.linear_e4m3(none, W).cpu(), torch.zeros(3, 64).bfloat16())
    got = ops.linear_e4m3(none, W, b.cuda(), "relu", r.cuda(), 0.5, torch.float32)
    assert torch.equal(got.cpu(), b.clamp_min(0) + 0.5 * r.float())


def test_lists_of_experts_that_share_their_ends():
    """Stacks belong to the very experts that were asked for: another list with the same first and last one, a part of a list, and the whole
    again, each gives what its experts give."""
    g = gen(5)
    a, b, c, d = [(on(whole(g, 256, 128)), on(whole(g, 128, 128))) for _ in range(4)]
    q = whole_rows(g, 9, 128)
    idx, w = torch.arange(9, dtype=torch.int32).view(9, 1) % 3, torch.ones(9, 1)
    first = [a, b, c]
    kept = ops.pack_experts_e4m3(first)
    for experts in (first, [a, d, c], [b, c, a], [a, b], first):
        want, tol = experts64(q, idx, w, experts)
        got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), experts, "relu")
        assert bool(((got.cpu().double() - want).abs() <= tol + 3 * 2.0 ** -24 * want.abs().amax(1, keepdim=True)).all())
    assert ops.pack_experts_e4m3(first) is kept
    check_status()


def test_copies_of_weights_and_captured_graphs():
    """A copy that a graph makes of a weight with odd rows is the graph's own; stacks are made before a capture or not at all."""
    from xfastertransformer_b200.ops import native as N
    g = gen(6)
    host = weight(g, 64, 200)
    W, x = on(host), activations(g, 3, 200).cuda()
    assert W.w.stride(0) % 16
    ops.quantize_e4m3(x)
    stream = torch.cuda.Stream()
    q = ops.quantize_e4m3(x)
    ops.linear_e4m3(q, on(host))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = ops.linear_e4m3(q, W)
    eager = ops.linear_e4m3(q, W)                                   # before the graph's copy has been made once
    graph.replay()
    want, tol = sum_tol(q, host)
    for got in (eager, y):
        assert bool(((got.cpu().double() - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all())
    experts = [(on(whole(g, 256, 128)), on(whole(g, 128, 128)))]
    qe, idx, w = rows_on(whole_rows(g, 2, 128)), torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(N.KernelError, match="before a graph"):
            ops.moe_experts_e4m3(qe, idx, w, experts, "relu")
        ops.linear_e4m3(q, W)
    check_status()


@pytest.mark.parametrize("T", [20, 100, 300])
def test_rows_that_are_not_finite_stay_alone(T):
    g = gen(T)
    x, W = torch.randn(T, 264, generator=g).bfloat16().cuda(), on(weight(g, 256, 264))
    want, wg = ops.linear_e4m3(ops.quantize_e4m3(x), W), ops.linear_gated_e4m3(ops.quantize_e4m3(x), W)
    x[3, 5], x[7, 200], x[9, 263] = float("inf"), float("nan"), float("-inf")
    got, gg = ops.linear_e4m3(ops.quantize_e4m3(x), W), ops.linear_gated_e4m3(ops.quantize_e4m3(x), W)
    keep = [i for i in range(T) if i not in (3, 7, 9)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[[3, 7, 9]]).all()
    assert torch.equal(gg.codes.view(torch.uint8)[keep], wg.codes.view(torch.uint8)[keep]) and torch.isnan(gg.codes.float()[[3, 7, 9]]).all()


@pytest.mark.parametrize("T", [9, 150])
def test_rows_and_weights_as_they_lie(T):
    """Codes and scales that are parts of wider tensors, between 16 bytes, or weights on an odd pitch: the bits of copies."""
    g = gen(T)
    q, W = rows_on(rows(torch.randn(T, 400, generator=g))), on(weight(g, 264, 400))
    want = ops.linear_e4m3(q, W, out_dtype=torch.float32)
    for at in (0, 3, 16):
        wide = torch.zeros(T, 450, dtype=torch.uint8, device="cuda")
        wide[:, at:at + 400] = q.codes.view(torch.uint8)
        scales = torch.zeros(4, T + 5, device="cuda")
        scales[:, 2:2 + T] = q.scale
        part = ops.RowsE4M3(wide.view(torch.float8_e4m3fn)[:, at:at + 400], scales[:, 2:2 + T])
        assert torch.equal(ops.linear_e4m3(part, W, out_dtype=torch.float32), want)
        assert torch.equal(ops.linear_e4m3(ops.RowsE4M3(q.codes, q.scale.t().contiguous().t()), W, out_dtype=torch.float32), want)
        ww = torch.zeros(264, 413, dtype=torch.uint8, device="cuda")
        ww[:, :400] = W.w.view(torch.uint8)
        V = LinearWeight("fp8a", ww.view(torch.float8_e4m3fn)[:, :400], W.scale, in_features=400, out_features=264)
        assert torch.equal(ops.linear_e4m3(q, V, out_dtype=torch.float32), want)
    for cols in (300, 301):
        out = torch.randn(T, cols, generator=g).bfloat16().cuda()
        for at in (0, 1, 4):
            res = out[:, at:at + 264]
            assert torch.equal(ops.linear_e4m3(q, W, None, None, res, 0.5), ops.linear_e4m3(q, W, None, None, res.clone(), 0.5))
    check_status()


def test_captured_and_on_another_stream():
    """The chain of a feed-forward layer, captured once and replayed on new inputs while another stream runs the same calls eagerly."""
    g = gen(3)
    T, H, I = 24, 512, 640
    x, r, gain = (torch.randn(T, H, generator=g).bfloat16().cuda() for _ in range(2)), None, torch.ones(H).cuda()
    xa, xb = x
    gu, dn = on(weight(g, 2 * I, H)), on(weight(g, H, I))

    def layer(v):
        q, _, h = ops.rmsnorm_e4m3(v, gain, 1e-6, v)
        return ops.linear_e4m3(ops.linear_gated_e4m3(q, gu), dn, residual=h)

    want = [layer(xa).clone(), layer(xb).clone()]
    static = xa.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(static)
    for i, v in enumerate((xb, xa, xb)):
        static.copy_(v)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other = layer(xa)
        torch.cuda.synchronize()
        assert torch.equal(out, want[(i + 1) % 2]) and torch.equal(other, want[0])
    check_status()


@pytest.mark.parametrize("T", [1, 50, 400])
def test_same_bits_every_time(T):
    g = gen(T)
    q, W = rows_on(rows(torch.randn(T, 2048, generator=g))), on(weight(g, 1024, 2048))
    first, second = ops.linear_gated_e4m3(q, W), ops.linear_e4m3(q, W)
    for _ in range(3):
        again = ops.linear_gated_e4m3(q, W)
        assert torch.equal(again.codes.view(torch.uint8), first.codes.view(torch.uint8)) and torch.equal(again.scale, first.scale)
        assert torch.equal(ops.linear_e4m3(q, W), second)


def test_refusals_of_the_kernels():
    from xfastertransformer_b200.ops.native import KernelError
    x = torch.zeros(2, 132, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError, match="multiple of 8"):
        ops.quantize_e4m3(x)
    with pytest.raises(KernelError, match="bf16"):
        ops.quantize_e4m3(torch.zeros(2, 128, device="cuda"))
    with pytest.raises(KernelError, match="32768"):
        ops.quantize_e4m3(torch.zeros(1, 32776, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(KernelError, match="residual"):
        ops.rmsnorm_e4m3(x[:, :128], torch.ones(128, device="cuda"), 1e-6, x[:, :128].half())
    q, W = ops.quantize_e4m3(x[:, :128]), on(weight(gen(1), 128, 128))
    with pytest.raises(KernelError, match="residual"):
        ops.linear_e4m3(q, W, residual=torch.zeros(2, 128, device="cuda"))
    with pytest.raises(ValueError, match="tensors on"):
        ops.linear_e4m3(q, W.to("cpu"))
