"""GPU: the operators over token rows -- quantisation, the int8 product with token and channel scales, products grouped
by expert and their gradients -- through the package's entry points, against plain implementations in 64 bits.

Tolerances.  Integer-valued data have exact sums, so results must equal the 64-bit value rounded once.  On real-valued
data a sum of K products of 16-bit values (exact in f32) or f32 values (each rounded: one more 2^-24) in any order is off
by at most (K + 1) * 2^-23 * S, S the sum of the products' magnitudes (half a step is 2^-24; the matrix instructions
are allowed a whole one), and the narrowing adds half a step of the result's type."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FLOATS = ("f16", "bf16", "f32")


def generator(seed):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return g


def whole(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g)


def _device_only(gpu):
    if gpu.type != "cuda":     # (the CPU build of the kernels in place of the device: kernel_host/as_device.py)
        pytest.skip("streams, graphs and gigabytes are not the model's business")


def make_offsets(sizes):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32))


def spans(sizes):
    ends = np.cumsum(sizes)
    return [(e, int(b - n), int(b)) for e, (n, b) in enumerate(zip(sizes, ends))]


def check_sum(got, exact, magnitude, depth, what=""):
    """`got` against the 64-bit sum `exact` of `depth` products whose magnitudes add up to `magnitude`."""
    got64 = got.double().cpu()
    tol = (depth + 1) * 2.0 ** -23 * magnitude
    half = torch.finfo(got.dtype).eps / 2
    tol = tol + half * (exact.abs() + tol) + torch.finfo(got.dtype).tiny * half
    bad = (got64 - exact).abs() > tol
    assert not bad.any(), (what, bad.nonzero()[0].tolist(), float((got64 - exact).abs().max()))


# ---- quantisation -------------------------------------------------------------------------------------------
def quantise64(x):
    """The definition: q and the scale, f32(max) / 127 rounded once."""
    x = x.detach().cpu().double().reshape(-1, x.shape[-1])
    top = x.abs().amax(dim=1)
    bad = ~torch.isfinite(x).all(dim=1)
    unit = torch.where(bad | (top == 0), 1.0, top)
    q = torch.where(bad[:, None], 0.0, torch.round(127.0 * torch.where(bad[:, None], 0.0, x) / unit[:, None]))
    scale = torch.from_numpy(top.float().numpy() / np.float32(127.0))
    scale[bad] = float("nan")
    return q.to(torch.int8), scale


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (7, 33), (3, 4095), (1500, 130), (1029, 8192), (2, 50000), (4000, 17)])
def test_quantize_tokens(rock, gpu, t, rows, cols):
    g = generator(rows + cols)
    x = torch.randn((rows, cols), generator=g) * torch.exp(torch.rand((rows, 1), generator=g) * 6 - 3)
    if rows > 5:
        x[1] = whole(g, -254, 254, cols).float()
        x[1, 0] = 254.0                # odd values are halves of a step
        x[2] = 0
        x[3, cols - 1] = float("-inf")
        x[4, cols // 2] = float("nan")
        x[5] *= 1e-38 if t == "f32" else 1e-6
    x = x.to(TORCH[t]).to(gpu)
    q, s = rock.quantize_tokens(x)
    want_q, want_s = quantise64(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (rows,)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(s.cpu().view(torch.int32)[~want_s.isnan()], want_s.view(torch.int32)[~want_s.isnan()])
    assert torch.equal(s.cpu().isnan(), want_s.isnan())


def test_quantize_tokens_of_views(rock, gpu):
    """Three dimensions, a column slice, a transposed tensor, a slice that starts off a 16-byte boundary, no rows,
    no columns, results written into given tensors."""
    g = generator(3)
    base = torch.randn((6, 40, 90), generator=g).to(torch.bfloat16).to(gpu)
    for x in (base, base[:, ::2, 3:80], base.transpose(1, 2), base.view(-1)[1:91], base[:0]):
        q, s = rock.quantize_tokens(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        if x.numel():
            want_q, want_s = quantise64(x.contiguous())
            assert torch.equal(q.cpu().reshape(want_q.shape), want_q) and torch.equal(s.cpu().reshape(-1), want_s)
    q, s = rock.quantize_tokens(base[0, :, :0])
    assert q.shape == (40, 0) and (s == 0).all()
    q_out, s_out = torch.empty((40, 90), dtype=torch.int8, device=gpu), torch.empty(40, device=gpu)
    q, s = rock.quantize_tokens(base[0], out=q_out, scale_out=s_out)
    assert q is q_out and s is s_out and torch.equal(q.cpu(), quantise64(base[0])[0])


# ---- int8 product with token and channel scales ---------------------------------------------------------------
def scaled64(acc, zp, channel, token, bias):
    """(acc - zp) * channel * token + bias as the kernels form it: one f32 operation per step (numpy's are IEEE)."""
    v = (acc.numpy().astype(np.float32) - np.float32(zp)) * channel.numpy()[None, :]
    v = v * token.numpy()[:, None]
    return torch.from_numpy(v if bias is None else v + bias.numpy()[None, :])


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("m,n,k,transB", [(1, 1, 1, True), (1, 4096, 512, True), (3, 129, 77, False), (16, 640, 1280, True), (17, 100, 400, True),
                                          (33, 72, 4096, True), (64, 257, 144, True), (65, 48, 80, False), (300, 515, 272, True), (520, 390, 2048, True),
                                          (300, 400, 336, False), (2000, 304, 64, True)])
def test_int8_product_with_token_scales(rock, gpu, out, m, n, k, transB):
    g = generator(m + n + k)
    a, b = whole(g, -128, 127, m, k).to(torch.int8), whole(g, -128, 127, n, k).to(torch.int8)
    token, channel = torch.rand(m, generator=g) * 0.01 + 0.001, torch.rand(n, generator=g) * 0.01 + 0.001
    bias = torch.randn(n, generator=g)
    acc = a.double() @ b.double().t()
    bd = (b if transB else b.t().contiguous()).to(gpu)
    got = rock.gemm(a.to(gpu), bd, transB=transB, out_dtype=out, scale=channel.to(gpu), token_scale=token.to(gpu))
    assert got.dtype == TORCH[out] and torch.equal(got.cpu(), scaled64(acc, 0, channel, token, None).to(TORCH[out]))
    got = rock.gemm(a.to(gpu), bd, transB=transB, out_dtype=out, scale=0.03125, zero_point=7, bias=bias.to(gpu), relu=True,
                    token_scale=token.to(gpu))
    want = scaled64(acc, 7, torch.full((n,), 0.03125), token, bias).clamp_min(0)
    assert torch.equal(got.cpu(), want.to(TORCH[out]))


def test_a_poisoned_token_poisons_its_own_row(rock, gpu):
    """An infinity or a NaN among the activations: the row of the product is NaN, the others are untouched."""
    g = generator(5)
    x = torch.randn((40, 256), generator=g).to(torch.float16)
    w = whole(g, -127, 127, 96, 256).to(torch.int8).to(gpu)
    x[7, 3] = float("inf")
    x[30, 200] = float("nan")
    q, s = rock.quantize_tokens(x.to(gpu))
    y = rock.gemm(q, w, transB=True, token_scale=s).cpu()
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[7, 30]] = True
    assert y[bad].isnan().all() and y[~bad].isfinite().all()
    for kw in (dict(relu=True), dict(clip=(-1.0, 1.0))):      # a clamp leaves a NaN alone, few rows or many
        for rows in (slice(0, 8), slice(0, 40)):
            y = rock.gemm(q[rows], w, transB=True, token_scale=s[rows], **kw).cpu()
            assert y[bad[rows]].isnan().all() and y[~bad[rows]].isfinite().all()
    off = make_offsets([8, 0, 32]).to(gpu)
    y = rock.grouped_gemm(q, w.expand(3, 96, 256), off, transB=True, token_scale=s).cpu()
    assert y[bad].isnan().all() and y[~bad].isfinite().all()


# ---- products grouped by expert ---------------------------------------------------------------------------------
CASES = [  # (rows per expert, rows behind the last, N, K)
    ([1], 0, 64, 64), ([7], 0, 100, 36), ([0, 5, 0, 1, 33, 0], 3, 130, 64), ([300, 0, 77, 128], 20, 264, 192),
    ([3] * 40 + [0] * 30 + [1] * 90, 5, 48, 80), ([0, 0, 0], 6, 32, 32), ([257, 255, 256], 1, 520, 1040),
    ([19, 45], 0, 33, 35), ([2, 1, 0, 9], 2, 768, 4096), ([64, 1], 0, 65, 72), ([1000], 0, 80, 16),
    ([130, 0, 290], 2, 75, 133), ([200, 0, 70], 1, 5, 3), ([1, 200], 0, 9, 131), ([90, 1, 200], 0, 300, 1002)]


def _ids(c):
    return "%dx%d-%d-%d" % (len(c[0]), sum(c[0]), c[2], c[3])


def grouped_operands(case, t, transB, integers, seed):
    sizes, tail, n, k = case
    g = generator(seed + sum(sizes) + n)
    T, E = sum(sizes) + tail, len(sizes)
    def draw(*shape):
        v = whole(g, -2, 2, *shape).float() if integers else torch.randn(shape, generator=g)
        return v.to(TORCH[t])
    x, w, dout = draw(T, k), draw(E, n, k), draw(T, n)
    for rows in (x, dout):            # rows of no expert are read by nothing
        rows[sum(sizes):] = float("nan")
    return g, T, E, x, (w if transB else w.transpose(1, 2).contiguous()), dout, make_offsets(sizes)


@pytest.mark.parametrize("integers", [True, False], ids=["integers", "reals"])
@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_grouped_gemm_and_its_gradients(rock, gpu, case, t, transB, integers):
    sizes, tail, n, k = case
    g, T, E, x, w, dout, off = grouped_operands(case, t, transB, integers, 11)
    d = [v.to(gpu) for v in (x, w, dout, off)]
    y = torch.full((T, n), -7.0, dtype=TORCH[t], device=gpu)
    dx = torch.full((T, k), -7.0, dtype=TORCH[t], device=gpu)
    assert rock.grouped_gemm(d[0], d[1], d[3], transB=transB, out=y) is y
    rock.grouped_gemm_bwd_data(d[2], d[1], d[3], transB=transB, out=dx)
    dw = rock.grouped_gemm_bwd_weight(d[0], d[2], d[3], transB=transB)
    assert dw.shape == w.shape and dw.dtype == w.dtype
    for e, a, b in spans(sizes):
        x64, d64 = x[a:b].double(), dout[a:b].double()
        w64 = (w[e] if transB else w[e].t()).double()      # [N, K]
        gw = d64.t() @ x64 if transB else x64.t() @ d64
        mw = d64.abs().t() @ x64.abs() if transB else x64.abs().t() @ d64.abs()
        for what, got, exact, mag, depth in (("y", y[a:b], x64 @ w64.t(), x64.abs() @ w64.abs().t(), k),
                                             ("dx", dx[a:b], d64 @ w64, d64.abs() @ w64.abs(), n),
                                             ("dw", dw[e], gw, mw, b - a)):
            if integers:
                assert torch.equal(got.cpu(), exact.to(TORCH[t])), (what, e)
            else:
                check_sum(got, exact, mag, depth, (what, e))
    assert (y[sum(sizes):] == -7).all() and (dx[sum(sizes):] == -7).all(), "rows of no expert were written"


def test_gradients_against_differences(rock, gpu):
    """The product is linear in x and in w: with integer-valued f32 data <dout, f(x + u) - f(x - u)> / 2 is exactly
    <dx, u>, and the same for w."""
    case = ([5, 0, 40, 1], 0, 72, 48)
    g, T, E, x, w, dout, off = grouped_operands(case, "f32", True, True, 3)
    u, v = whole(g, -2, 2, *x.shape).float(), whole(g, -2, 2, *w.shape).float()
    x, w, dout, off, u, v = (t.to(gpu) for t in (x, w, dout, off, u, v))
    f = lambda x, w: rock.grouped_gemm(x, w, off, transB=True).double()   # noqa: E731
    dx, dw = rock.grouped_gemm_bwd_data(dout, w, off, transB=True), rock.grouped_gemm_bwd_weight(x, dout, off, transB=True)
    assert ((f(x + u, w) - f(x - u, w)) * dout).sum() / 2 == (dx.double() * u).sum()
    assert ((f(x, w + v) - f(x, w - v)) * dout).sum() / 2 == (dw.double() * v).sum()


TILES = ["16,16", "16,32", "32,16", "32,32", "64,64", "128,128", "256,256"]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("n,k", [(272, 208), (205, 131)], ids=["chunks", "any"])
@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
@pytest.mark.parametrize("t", FLOATS + ("i8",))
def test_every_kernel(rock, gpu, t, transB, n, k, tile):
    """Every tile of every product and gradient, by request: groups that end inside a tile, at its end and one row
    behind it, an empty one, rows of none.  Exact sums."""
    sizes, tail = [64, 0, 257, 129, 1, 16], 3
    g, T, E = generator(n + k), sum(sizes) + tail, len(sizes)
    kind = torch.int8 if t == "i8" else TORCH[t]
    x, w, dout = whole(g, -2, 2, T, k).to(kind), whole(g, -2, 2, E, n, k).to(kind), whole(g, -2, 2, T, n).to(kind)
    wd = (w if transB else w.transpose(1, 2).contiguous()).to(gpu)
    off, xd, dd = make_offsets(sizes).to(gpu), x.to(gpu), dout.to(gpu)
    perf, info = "v2:" + tile, {}
    y = torch.full((T, n), -7.0, dtype=torch.float32, device=gpu)
    rock.grouped_gemm(xd, wd, off, transB=transB, out_dtype="f32", out=y, perf_config=perf, info=info)
    if transB:      # (the kernels for few rows take weights stored [N, K] only, those of any alignment have no 256 x 256)
        assert tile.replace(",", "x") in info["kernel_name"] or (tile == "256,256" and "_any" in info["kernel_name"])
    for e, a, b in spans(sizes):
        assert torch.equal(y[a:b].cpu(), (x[a:b].double() @ w[e].double().t()).float()), (info, e)
    assert (y[sum(sizes):] == -7).all()
    if t == "i8":
        return
    dx = rock.grouped_gemm_bwd_data(dd, wd, off, transB=transB, perf_config=perf)
    dw = rock.grouped_gemm_bwd_weight(xd, dd, off, transB=transB, perf_config=perf)
    for e, a, b in spans(sizes):
        assert torch.equal(dx[a:b].cpu(), (dout[a:b].double() @ w[e].double()).to(kind)), e
        want = dout[a:b].double().t() @ x[a:b].double()
        assert torch.equal(dw[e].cpu(), (want if transB else want.t()).to(kind)), e


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("sizes", [[3000, 0, 33, 1], [64], [257, 512]], ids=str)
def test_weight_gradient_split_over_the_waves(rock, gpu, t, sizes):
    case = (sizes, 2, 136, 72)
    for integers in (True, False):
        g, T, E, x, w, dout, off = grouped_operands(case, t, True, integers, 17)
        info = {}
        dw = rock.grouped_gemm_bwd_weight(x.to(gpu), dout.to(gpu), off.to(gpu), transB=True, info=info,
                                          perf_config="v2:64,64,8,32,16,8,4,1,1")
        assert info["kernel_name"].endswith("_64x64_split")
        for e, a, b in spans(sizes):
            x64, d64 = x[a:b].double(), dout[a:b].double()
            check_sum(dw[e], d64.t() @ x64, d64.abs().t() @ x64.abs(), b - a, e)


@pytest.mark.parametrize("t,n,k", [("bf16", 2056, 72), ("f32", 1100, 40)])
def test_tiles_in_whole_rounds_and_parts(rock, gpu, t, n, k):
    """More 256 x 256 tiles than compute units in the product and both gradients, so that whole tiles, halves and
    quarters run in one launch."""
    sizes = [300, 1, 0, 2000, 513, 256, 40, 700]
    g, T, E = generator(n), sum(sizes), len(sizes)
    x, w, dout = (whole(g, -1, 1, *s).to(TORCH[t]).to(gpu) for s in ((T, k), (E, n, k), (T, n)))
    off = make_offsets(sizes).to(gpu)
    kw = dict(transB=True, perf_config="v2:256,256")
    y, dw = rock.grouped_gemm(x, w, off, **kw), rock.grouped_gemm_bwd_weight(x, dout, off, **kw)
    wide = rock.grouped_gemm_bwd_data(x, w.transpose(1, 2).contiguous(), off, **kw)     # as dout [T, k] of weights [E, k, n]
    for e, a, b in spans(sizes):
        want = (x[a:b].cpu().double() @ w[e].cpu().double().t()).to(TORCH[t])
        assert torch.equal(y[a:b].cpu(), want) and torch.equal(wide[a:b].cpu(), want), e
        assert torch.equal(dw[e].cpu(), (dout[a:b].cpu().double().t() @ x[a:b].cpu().double()).to(TORCH[t])), e


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_grouped_int8_product(rock, gpu, case, transB, out):
    sizes, tail, n, k = case
    g, T, E = generator(n + k), sum(sizes) + tail, len(sizes)
    x, w = whole(g, -128, 127, T, k).to(torch.int8), whole(g, -128, 127, E, n, k).to(torch.int8)
    token, channel = torch.rand(T, generator=g) * 0.01 + 0.001, torch.rand((E, n), generator=g) * 0.01 + 0.001
    wd = (w if transB else w.transpose(1, 2).contiguous()).to(gpu)
    xd, off, y = x.to(gpu), make_offsets(sizes).to(gpu), torch.full((T, n), -7.0, dtype=TORCH[out], device=gpu)
    rock.grouped_gemm(xd, wd, off, transB=transB, out_dtype=out, token_scale=token.to(gpu), scale=channel.to(gpu), out=y)
    plain = rock.grouped_gemm(xd, wd, off, transB=transB, out_dtype=out, scale=0.0078125)
    for e, a, b in spans(sizes):
        acc = x[a:b].double() @ w[e].double().t()
        assert torch.equal(y[a:b].cpu(), scaled64(acc, 0, channel[e], token[a:b], None).to(TORCH[out])), e
        assert torch.equal(plain[a:b].cpu(), (acc.float() * 0.0078125).to(TORCH[out])), e
    assert (y[sum(sizes):] == -7).all()


@pytest.mark.parametrize("t,out", [("f16", "f32"), ("bf16", "f16"), ("f32", "bf16")])
def test_grouped_gemm_result_of_another_type(rock, gpu, t, out):
    case = ([9, 0, 70], 2, 72, 128)
    g, T, E, x, w, dout, off = grouped_operands(case, t, True, True, 5)
    y = rock.grouped_gemm(x.to(gpu), w.to(gpu), off.to(gpu), transB=True, out_dtype=out)
    for e, a, b in spans(case[0]):
        assert torch.equal(y[a:b].cpu(), (x[a:b].double() @ w[e].double().t()).to(TORCH[out]))


def test_operands_that_are_views(rock, gpu):
    """Slices of rows and columns, weights as a transposed view, offsets out of the middle of a tensor."""
    case = ([6, 0, 31], 4, 64, 96)
    g, T, E, x, w, dout, off = grouped_operands(case, "bf16", True, True, 8)
    wide = torch.zeros((T + 1, 200), dtype=torch.bfloat16, device=gpu)
    wide[1:, 5:101] = x.to(gpu)
    longer = torch.cat([torch.full((3,), 99, dtype=torch.int32), off]).to(gpu)
    wt = w.transpose(1, 2).contiguous().to(gpu)       # [E, K, N]
    want = rock.grouped_gemm(x.to(gpu), w.to(gpu), off.to(gpu), transB=True)
    got = rock.grouped_gemm(wide[1:, 5:101], wt.transpose(1, 2), longer[3:], transB=True)
    assert torch.equal(got[:37], want[:37])


@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 2, 100, 7], [2147483647] * 4, [-2147483648, 1, 1, 12]])
def test_offsets_out_of_order_or_range(rock, gpu, offsets):
    """Read as the furthest boundary before them (checked against every tensor's bounds on the CPU build of the kernels,
    tests/test_token_ops_model.py)."""
    g = generator(1)
    x, w = whole(g, -2, 2, 12, 32).half(), whole(g, -2, 2, 3, 24, 32).half()
    y = torch.full((12, 24), -7.0, dtype=torch.float16, device=gpu)
    rock.grouped_gemm(x.to(gpu), w.to(gpu), torch.tensor(offsets, dtype=torch.int32, device=gpu), transB=True, out=y)
    at = np.maximum.accumulate(np.clip(np.asarray(offsets, np.int64), 0, 12))
    want = torch.full((12, 24), -7.0, dtype=torch.float16)
    for e in range(3):
        want[at[e]:at[e + 1]] = (x[at[e]:at[e + 1]].double() @ w[e].double().t()).half()
    assert torch.equal(y.cpu(), want)


def test_no_rows_at_all(rock, gpu):
    off = torch.zeros(3, dtype=torch.int32, device=gpu)
    x, w = torch.empty((0, 32), dtype=torch.float16, device=gpu), torch.randn((2, 16, 32), device=gpu).half()
    assert rock.grouped_gemm(x, w, off, transB=True).shape == (0, 16)
    dout = torch.empty((0, 16), dtype=torch.float16, device=gpu)
    assert rock.grouped_gemm_bwd_data(dout, w, off, transB=True).shape == (0, 32)
    assert (rock.grouped_gemm_bwd_weight(x, dout, off, transB=True) == 0).all()
    assert rock.gemm(torch.empty((0, 32), dtype=torch.int8, device=gpu), torch.ones((8, 32), dtype=torch.int8, device=gpu),
                     transB=True, token_scale=torch.empty(0, device=gpu)).shape == (0, 8)


def test_rows_behind_two_gibibytes(rock, gpu):
    """Rows whose byte positions pass 2^31 and 2^32, in the operands of the product and of both gradients."""
    _device_only(gpu)
    n, k, T = 2048, 32, 1_100_000                       # dout: 4.5 GB
    sizes = [520_000, 530_000, 49_990]                  # groups start at 2.1 GB and 4.3 GB of dout
    off = make_offsets(sizes).to(gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    x = torch.randint(-1, 2, (T, k), generator=g, device=gpu).half()
    w = torch.randint(-1, 2, (3, n, k), generator=g, device=gpu).half()
    y = torch.full((T, n), -7.0, dtype=torch.float16, device=gpu)
    rock.grouped_gemm(x, w, off, transB=True, out=y)
    for e, a, b in spans(sizes):
        for r in (slice(a, a + 300), slice(b - 300, b)):
            assert torch.equal(y[r], (x[r].float() @ w[e].float().t()).half())
    assert (y[sum(sizes):] == -7).all()
    dx = rock.grouped_gemm_bwd_data(y, w, off, transB=True)
    for e, a, b in spans(sizes):
        for r in (slice(a, a + 300), slice(b - 300, b)):
            want = (y[r].double().cpu() @ w[e].double().cpu()).half()
            assert torch.equal(dx[r].cpu(), want)       # sums of whole numbers below 2^24
    # few non-zero rows per group, the last one among them: sums stay exact
    keep = torch.zeros(T, dtype=torch.bool, device=gpu)
    for _, a, b in spans(sizes):
        keep[a:a + 5] = True
        keep[b - 5:b] = True
    x[~keep] = 0
    dw = rock.grouped_gemm_bwd_weight(x, y, off, transB=True)
    for e, a, b in spans(sizes):
        rows = torch.tensor(list(range(a, a + 5)) + list(range(b - 5, b)), device=gpu)
        want = y[rows].double().cpu().t() @ x[rows].double().cpu()
        assert torch.equal(dw[e].cpu(), want.half())


# ---- as they are used -------------------------------------------------------------------------------------------
def test_int8_experts_from_tokens_to_tokens(rock, gpu):
    """A quantised mixture layer: tokens quantised, sent through the experts' first product, gated, quantised again,
    sent through the second, and a dense int8 product behind it; every step against its definition on the step's own
    inputs."""
    sizes, hidden, inner = [3, 0, 40, 1, 20], 128, 208
    g, T, E = generator(21), 64, 5
    off = make_offsets(sizes).to(gpu)
    x = torch.randn((T, hidden), generator=g).to(torch.bfloat16).to(gpu)
    w1, w2 = whole(g, -127, 127, E, inner, hidden).to(torch.int8).to(gpu), whole(g, -127, 127, E, hidden, inner).to(torch.int8).to(gpu)
    s1, s2 = (torch.rand((E, inner), generator=g) * 1e-3).to(gpu), (torch.rand((E, hidden), generator=g) * 1e-3).to(gpu)
    wd, sd = whole(g, -127, 127, 96, hidden).to(torch.int8).to(gpu), (torch.rand(96, generator=g) * 1e-3).to(gpu)

    def step(x, w, s):
        q, t = rock.quantize_tokens(x)
        y = rock.grouped_gemm(q, w, off, transB=True, out_dtype="bf16", token_scale=t, scale=s)
        want_q, want_t = quantise64(x)
        assert torch.equal(q.cpu(), want_q) and torch.equal(t.cpu(), want_t)
        for e, a, b in spans(sizes):
            acc = want_q[a:b].double() @ w[e].cpu().double().t()
            assert torch.equal(y[a:b].cpu(), scaled64(acc, 0, s[e].cpu(), want_t[a:b], None).to(torch.bfloat16)), e
        return y
    h = step(x, w1, s1)
    h = (h.float() * torch.sigmoid(h.float())).to(torch.bfloat16)
    h = step(h, w2, s2)
    q, t = rock.quantize_tokens(h)
    y = rock.gemm(q, wd, transB=True, out_dtype="bf16", token_scale=t, scale=sd)
    want_q, want_t = quantise64(h)
    assert torch.equal(y.cpu(), scaled64(want_q.double() @ wd.cpu().double().t(), 0, sd.cpu(), want_t, None).to(torch.bfloat16))


def test_a_training_step_replayed_from_a_graph(rock, gpu):
    """Forward and both gradients of a grouped product, and a quantised product, captured once and replayed on new
    inputs, offsets included, with eager work between the replays: equal to the eager calls bit for bit."""
    _device_only(gpu)
    E, T, n, k = 6, 200, 136, 96
    g = generator(31)
    x, dout = torch.zeros((T, k), dtype=torch.bfloat16, device=gpu), torch.zeros((T, n), dtype=torch.bfloat16, device=gpu)
    w = torch.randn((E, n, k), generator=g).to(torch.bfloat16).to(gpu)
    wq = whole(g, -127, 127, n, k).to(torch.int8).to(gpu)
    off = torch.zeros(E + 1, dtype=torch.int32, device=gpu)
    y, dx = torch.zeros((T, n), dtype=torch.bfloat16, device=gpu), torch.zeros((T, k), dtype=torch.bfloat16, device=gpu)

    def work(y, dx):
        rock.grouped_gemm(x, w, off, transB=True, out=y)
        rock.grouped_gemm_bwd_data(dout, w, off, transB=True, out=dx)
        dw = rock.grouped_gemm_bwd_weight(x, dout, off, transB=True)
        q, s = rock.quantize_tokens(x)
        return y, dx, dw, q, s, rock.gemm(q, wq, transB=True, token_scale=s)
    work(y, dx)      # loads the code objects
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work(y, dx)
    for trial in range(4):
        x.copy_(torch.randn((T, k), generator=g).to(torch.bfloat16))
        dout.copy_(torch.randn((T, n), generator=g).to(torch.bfloat16))
        counts = np.random.default_rng(trial).multinomial(T - 3 * trial, np.full(E, 1 / E))
        off.copy_(make_offsets(counts))
        y.zero_()
        dx.zero_()
        graph.replay()
        eager = work(torch.zeros_like(y), torch.zeros_like(dx))
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_streams_and_threads(rock, gpu):
    """The same problem from two threads on streams of their own, operands made on those streams; and a stream passed
    by argument, as an object and as a raw handle."""
    _device_only(gpu)
    g = generator(41)
    sizes, n, k = [50, 3, 90], 200, 160
    off = make_offsets(sizes).to(gpu)
    w = whole(g, -2, 2, 3, n, k).half().to(gpu)
    xs = [whole(g, -2, 2, 143, k).half().to(gpu) for _ in range(2)]
    want = [torch.cat([(x[a:b].float() @ w[e].float().t()).half() for e, a, b in spans(sizes)]) for x in xs]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def worker(i):
        try:
            torch.cuda.set_device(gpu)
            s = torch.cuda.Stream(device=gpu)
            with torch.cuda.stream(s):
                for _ in range(20):
                    x = xs[i] * 1
                    results[i] = rock.grouped_gemm(x, w, off, transB=True)
            s.synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert torch.equal(results[0], want[0]) and torch.equal(results[1], want[1])
    s = torch.cuda.Stream(device=gpu)
    for given in (s, s.cuda_stream):
        y = rock.grouped_gemm(xs[0], w, off, transB=True, stream=given)
        s.synchronize()
        assert torch.equal(y, want[0])


@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 2, 100, 7], [9, 0, 0, 0], [2147483647] * 4, [-2147483648, 1, 1, 12],
                                     [0, 40, 7] + [8] * 80 + [60, 2, 90] + [0] * 70 + [130, 5]], ids=lambda o: "-".join(map(str, o[:4])))
@pytest.mark.parametrize("n,k", [(24, 32), (21, 33)], ids=["chunks", "any"])
@pytest.mark.parametrize("t", FLOATS)
def test_gradients_on_offsets_out_of_order_or_range(rock, gpu, t, n, k, offsets):
    """The gradients read the boundaries as the product does (every address checked on the CPU build of the kernels first,
    tests/test_token_ops_model.py): no row counts in two groups, rows of none are left as they were."""
    T, E = 131, len(offsets) - 1
    g = generator(2)
    x, w, dout = (whole(g, -2, 2, *s).to(TORCH[t]) for s in ((T, k), (E, n, k), (T, n)))
    off = torch.tensor(offsets, dtype=torch.int32, device=gpu)
    at = np.maximum.accumulate(np.clip(np.asarray(offsets, np.int64), 0, T))
    for perf in (None, "v2:64,64,8,32,16,8,4,1,1", "v2:128,128", "v2:256,256"):
        dw = rock.grouped_gemm_bwd_weight(x.to(gpu), dout.to(gpu), off, transB=True, perf_config=perf).cpu()
        for e in range(E):
            a, b = at[e], at[e + 1]
            assert torch.equal(dw[e], (dout[a:b].double().t() @ x[a:b].double()).to(TORCH[t])), (perf, e)
    dx = torch.full((T, k), -7.0, dtype=TORCH[t], device=gpu)
    rock.grouped_gemm_bwd_data(dout.to(gpu), w.to(gpu), off, transB=True, out=dx)
    want = torch.full((T, k), -7.0, dtype=TORCH[t])
    for e in range(E):
        want[at[e]:at[e + 1]] = (dout[at[e]:at[e + 1]].double() @ w[e].double()).to(TORCH[t])
    assert torch.equal(dx.cpu(), want)


def test_the_default_stream_by_its_handle(rock, gpu):
    """The raw handle of the default stream is 0: such a call is ordered with the work queued there, also while another
    stream is the current one."""
    _device_only(gpu)
    import rocmlir_amd.api as api
    default, side = torch.cuda.default_stream(gpu), torch.cuda.Stream(device=gpu)
    assert default.cuda_stream == 0
    g = generator(43)
    src = torch.randn((4000, 2048), generator=g).half().to(gpu)
    want_q, want_s = quantise64(src)
    x, big = torch.zeros_like(src), torch.randn((4096, 4096), generator=g).to(gpu)
    torch.cuda.synchronize()
    for given in (0, default):
        with torch.cuda.stream(side):
            with api._on("test", gpu, given):
                assert torch.cuda.current_stream() == default
        x.zero_()
        for _ in range(4):
            big @ big                  # the copy waits behind these
        x.copy_(src)
        with torch.cuda.stream(side):
            q, s = rock.quantize_tokens(x, stream=given)
        default.synchronize()
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_single_rows_longer_than_two_gibibytes(rock, gpu, t):
    """Columns whose byte position in their row passes 2^31, of weights stored [K, N] and of activations (every address
    checked on the CPU build of the kernels first, tests/test_token_ops_model.py)."""
    _device_only(gpu)
    es = 2 if t == "f16" else 4
    wide, depth, g = (1 << 31) // es + 203, 9, generator(47)
    places = [slice(0, 300), slice(wide // 2 - 150, wide // 2 + 150), slice(wide - 203 - 300, wide - 203), slice(wide - 300, wide)]
    long_rows = torch.zeros((depth, wide), dtype=TORCH[t], device=gpu)
    for p in places:
        long_rows[:, p] = whole(g, -3, 3, depth, 300).to(TORCH[t]).to(gpu)
    x = whole(g, -3, 3, 2, depth).to(TORCH[t])
    y = rock.grouped_gemm(x.to(gpu), long_rows[None], torch.tensor([0, 2], dtype=torch.int32, device=gpu))
    dy = whole(g, -3, 3, depth, 9).to(TORCH[t])
    dw = rock.grouped_gemm_bwd_weight(long_rows, dy.to(gpu), torch.tensor([0, depth], dtype=torch.int32, device=gpu))
    for p in places:
        cols = long_rows[:, p].cpu().double()
        assert torch.equal(y[:, p].cpu().double(), x.double() @ cols), p
        assert torch.equal(dw[0, p].cpu().double(), cols.t() @ dy.double()), p
    assert not y[:, 300:700].any() and not dw[0, 300:700].any()


@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
def test_a_reduction_over_nothing(rock, gpu, transB):
    """K = 0 (N = 0 in the gradient of the rows): sums of nothing are 0, the epilogue is applied to them, and rows of no
    expert stay as they were.  What quantize_tokens returns for rows without elements goes through the products."""
    off = make_offsets([2, 0, 3]).to(gpu)
    x = torch.empty((7, 0), dtype=torch.bfloat16, device=gpu)
    w = torch.empty((3, 6, 0) if transB else (3, 0, 6), dtype=torch.bfloat16, device=gpu)
    y = torch.full((7, 6), -7.0, dtype=torch.bfloat16, device=gpu)
    rock.grouped_gemm(x, w, off, transB=transB, out=y)
    assert (y[:5] == 0).all() and (y[5:] == -7).all()
    wd = torch.empty((3, 0, 6) if transB else (3, 6, 0), dtype=torch.bfloat16, device=gpu)
    dx = torch.full((7, 6), -7.0, dtype=torch.bfloat16, device=gpu)
    rock.grouped_gemm_bwd_data(x, wd, off, transB=transB, out=dx)
    assert (dx[:5] == 0).all() and (dx[5:] == -7).all()
    q, s = rock.quantize_tokens(x)
    assert q.shape == (7, 0) and (s == 0).all()
    wq = torch.empty((3, 6, 0) if transB else (3, 0, 6), dtype=torch.int8, device=gpu)
    y = torch.full((7, 6), -7.0, dtype=torch.float16, device=gpu)
    rock.grouped_gemm(q, wq, off, transB=transB, token_scale=s, scale=torch.ones((3, 6), device=gpu), out=y)
    assert (y[:5] == 0).all() and (y[5:] == -7).all()
    token, bias = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0, 6.0, float("nan")], device=gpu), torch.arange(6.0, device=gpu)
    y = rock.gemm(q, wq[0], transB=transB, token_scale=token, scale=0.5, zero_point=3, bias=bias, out_dtype="f32")
    want = -1.5 * token[:, None] + bias
    assert torch.equal(y[:6], want[:6]) and y[6].isnan().all()


# (rows per expert, N, K): 256 x 256 tiles of the product, of the gradient of the rows and of the weights'
ROUNDS = [([300, 1, 0, 2000, 513, 256, 40, 700], 4064, 4112, "quarters"),    # 19 row tiles x 16: 256 + 48; x 17: 256 + 67 (halves)
          ([300, 1, 0, 2000, 513, 256, 40, 700], 4592, 4096, "halves"),      # x 18: 256 + 86; x 16: 256 + 48 (quarters)
          ([700, 0, 33], 2832, 3600, "weights")]                             # 3 x 12 x 15: 512 + 28; dW alone passes a round


@pytest.mark.parametrize("t", ["bf16", "i8"])
@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
@pytest.mark.parametrize("sizes,n,k,which", ROUNDS, ids=[r[3] for r in ROUNDS])
def test_whole_rounds_of_tiles_and_then_parts(rock, gpu, sizes, n, k, which, transB, t):
    """More 256 x 256 tiles than compute units: whole rounds of them, then what is left in quarters (up to 64 tiles) or in
    halves (up to 128), in the product, the gradient of the rows and the gradient of the weights."""
    _device_only(gpu)
    tiles = lambda c: -(-c // 256)   # noqa: E731
    rows, E, T = sum(tiles(s) for s in sizes), len(sizes), sum(sizes)
    of_products, of_weights = (rows * tiles(n), rows * tiles(k)), E * tiles(n) * tiles(k)
    counted = of_products if which != "weights" else (of_weights,)
    assert all(c > 256 and 0 < c % 256 <= 128 for c in counted), (of_products, of_weights)
    assert which == "weights" or {c % 256 <= 64 for c in counted} == {True, False}     # quarters in one, halves in the other
    kind, g = torch.int8 if t == "i8" else TORCH[t], torch.Generator(device=gpu)
    g.manual_seed(n)
    # 40 columns of x and of dout are not 0, so that the 64-bit products here stay short; they sum exactly
    some_k, some_n = (torch.randperm(c, generator=generator(c))[:40].sort().values.to(gpu) for c in (k, n))
    x, dout = torch.zeros((T, k), dtype=kind, device=gpu), torch.zeros((T, n), dtype=kind, device=gpu)
    x[:, some_k] = torch.randint(-2, 3, (T, 40), generator=g, device=gpu).to(kind)
    dout[:, some_n] = torch.randint(-2, 3, (T, 40), generator=g, device=gpu).to(kind)
    w = torch.randint(-1, 2, (E, n, k), generator=g, device=gpu, dtype=torch.int8).to(kind)
    wd, off = (w if transB else w.transpose(1, 2).contiguous()), make_offsets(sizes).to(gpu)
    info, kw = {}, dict(transB=transB, perf_config="v2:256,256")
    y = rock.grouped_gemm(x, wd, off, out_dtype="f32" if t == "i8" else None, info=info, **kw)
    assert "256x256_fast" in info["kernel_name"]
    if t != "i8":
        dx, dw = rock.grouped_gemm_bwd_data(dout, wd, off, **kw), rock.grouped_gemm_bwd_weight(x, dout, off, info=info, **kw)
        assert info["kernel_name"].endswith("256x256")
    for e, a, b in spans(sizes):
        xe, de, we = x[a:b][:, some_k].double(), dout[a:b][:, some_n].double(), w[e].double()
        assert torch.equal(y[a:b], (xe @ we[:, some_k].t()).to(y.dtype)), e
        if t != "i8":
            assert torch.equal(dx[a:b], (de @ we[some_n]).to(kind)), e
            want = torch.zeros((n, k), dtype=torch.float64, device=gpu)
            want[some_n[:, None], some_k] = de.t() @ xe
            assert torch.equal(dw[e], (want if transB else want.t()).to(kind)), e


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("n,k", [(72, 80), (69, 77)], ids=["chunks", "any"])
@pytest.mark.parametrize("transB", [True, False], ids=["NK", "KN"])
@pytest.mark.parametrize("t", FLOATS)
def test_what_is_not_finite_stays_in_its_row_and_column(rock, gpu, t, transB, n, k, tile):
    """A NaN in a row of x, an infinity in a column of one expert's weights: what the 64-bit products hold, nothing in the
    rows and experts beside them, in the product and in both gradients."""
    sizes, tail = [30, 0, 70, 1], 2
    g, T, E, x, w, dout, off = grouped_operands((sizes, tail, n, k), t, True, True, 23)
    x[5, k - 1], w[2, n - 1, 3], dout[40, 2], x[29, 0] = float("nan"), float("inf"), float("inf"), float("-inf")
    wd = (w if transB else w.transpose(1, 2).contiguous()).to(gpu)
    xd, dd, offd, kw = x.to(gpu), dout.to(gpu), off.to(gpu), dict(transB=transB, perf_config="v2:" + tile)
    y, dx = rock.grouped_gemm(xd, wd, offd, **kw).cpu(), rock.grouped_gemm_bwd_data(dd, wd, offd, **kw).cpu()
    dw = rock.grouped_gemm_bwd_weight(xd, dd, offd, **kw).cpu()
    same = lambda got, want: torch.equal(got.double().nan_to_num(nan=9e9), want.to(TORCH[t]).double().nan_to_num(nan=9e9))   # noqa: E731
    for e, a, b in spans(sizes):
        x64, d64, w64 = x[a:b].double(), dout[a:b].double(), w[e].double()
        assert same(y[a:b], x64 @ w64.t()) and same(dx[a:b], d64 @ w64), e
        assert same(dw[e], d64.t() @ x64 if transB else x64.t() @ d64), e


@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("rows,k", [(3, 256), (40, 256), (40, 77), (600, 256)])
def test_poisoned_tokens_in_every_result_type(rock, gpu, out, rows, k):
    g = generator(51)
    x = torch.randn((rows, k), generator=g).to(torch.bfloat16)
    x[rows // 2, 1] = float("inf")
    w = whole(g, -127, 127, 96, k).to(torch.int8)
    q, s = rock.quantize_tokens(x.to(gpu))
    for trans in (True, False):
        wd = (w if trans else w.t().contiguous()).to(gpu)
        for y in (rock.gemm(q, wd, transB=trans, token_scale=s, out_dtype=out, relu=True),
                  rock.grouped_gemm(q, wd[None], make_offsets([rows]).to(gpu), transB=trans, token_scale=s, out_dtype=out)):
            bad = torch.arange(rows, device=gpu) == rows // 2
            assert y[bad].isnan().all() and y[~bad].isfinite().all()
