"""The kernels over token rows (csrc/token_gemm.h, csrc/quantize_tokens.hip) built for the CPU and run through whole
plans: every address checked, loads landing at issue or at their wait, no byte written by two blocks, and on
integer-valued data results equal to numpy's bit for bit.  The plans come from the C ABI as a caller gets them."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tests.kernel_host.model import CLANG, build_model, pointer_map, run_plan  # noqa: E402

pytestmark = pytest.mark.skipif(CLANG is None, reason="the host build uses clang's vector extensions")

_NUMPY = {"f32": np.float32, "f16": np.float16, "i8": np.int8}


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    lib = build_model(str(tmp_path_factory.mktemp("kernel_host_tokens")), types=(), attention=False, tokens=(0, 1, 3))
    lib.hm_set_owner_check(1)
    return lib


@pytest.fixture(params=["loads-land-at-issue", "loads-land-at-the-wait"])
def loads(request, model):
    late = request.param == "loads-land-at-the-wait"
    model.hm_set_late_loads(1 if late else 0)
    model.hm_set_thread_order(2 if late else 0)
    yield request.param
    model.hm_set_late_loads(0)
    model.hm_set_thread_order(0)


@pytest.fixture(scope="module")
def rock():
    import rocmlir_amd
    rocmlir_amd.load_library()
    return rocmlir_amd


def bounds(offsets, T):
    """The groups' rows as the operators read them: offsets clamped to the rows, none before one in front of it."""
    at = np.maximum.accumulate(np.clip(np.asarray(offsets, np.int64), 0, T))
    return list(zip(at[:-1], at[1:]))


def flag(b):
    return str(bool(b)).lower()


# ---- quantisation ---------------------------------------------------------------------------------------------
def quantise_reference(x):
    """The definition in 64 bits: roundeven(127 x / max), and max / 127 rounded to f32 once."""
    x = x.astype(np.float64)
    top = np.abs(x).max(axis=1)
    bad = ~np.isfinite(x).all(axis=1)
    unit = np.where(bad | (top == 0), 1.0, top)
    q = np.where(bad[:, None], 0.0, np.rint(127.0 * np.where(bad[:, None], 0.0, x) / unit[:, None])).astype(np.int8)
    scale = (top.astype(np.float32) / np.float32(127.0)).astype(np.float32)
    scale[bad] = np.nan
    return q, scale


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (9, 513), (1030, 24), (2, 4100), (1027, 4104), (1, 20000)])
def test_quantisation_equals_the_definition(model, rock, t, rows, cols):
    rng = np.random.default_rng(rows * 31 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-3, 3, (rows, 1)))).astype(_NUMPY[t])
    # ties: whole and half steps of a row whose largest magnitude is 127 (or 254, where odd values are halves)
    x[0] = (rng.integers(-254, 255, cols)).astype(_NUMPY[t])
    x[0, 0] = 254
    if rows > 2:
        x[1] = 0
        x[2, cols // 2] = np.inf
    if rows > 4:
        x[3, cols - 1] = np.nan
        x[4] = x[4] * _NUMPY[t](1e-6)      # f16: subnormal
    if rows > 8 and t == "f32":
        x[5] = (x[5].astype(np.float64) * 1e-38).astype(np.float32)   # 127 / max overflows
        x[6] = (x[6].astype(np.float64) * 1e36).astype(np.float32)
    names, problems, out = run_plan(model, rock, "-operation quantize_tokens -t %s -m %d -k %d" % (t, rows, cols), {0: x})
    assert names == ["rock_quantize_tokens_" + t] and not problems, (names, problems)
    q, scale = quantise_reference(x)
    assert np.array_equal(out[1][:q.size].view(np.int8).reshape(q.shape), q)
    assert np.array_equal(out[2][:4 * rows].view(np.float32), scale, equal_nan=True)


# ---- int8 product with token and channel scales -----------------------------------------------------------------
def scaled(acc, zp, channel, token, bias, out):
    """The epilogue, one f32 operation per step."""
    v = (acc.astype(np.float32) - np.float32(zp)) * channel.astype(np.float32)
    v = (v * token[:, None].astype(np.float32)).astype(np.float32)
    if bias is not None:
        v = v + bias[None, :].astype(np.float32)
    return v.astype(_NUMPY[out])


@pytest.mark.parametrize("shape,transB,extra", [
    ((1, 64, 128), True, ""), ((70, 45, 96), True, ""), ((33, 40, 100), True, ""), ((50, 48, 64), False, ""),
    ((20, 33, 48), False, ""), ((300, 260, 144), True, "-perf_config v2:256,256"), ((130, 200, 272), True, "-perf_config v2:128,128"),
    ((130, 208, 80), False, "-perf_config v2:128,128"), ((260, 272, 160), False, "-perf_config v2:256,256")],
    ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
@pytest.mark.parametrize("out,vector,bias", [("f16", True, True), ("f32", False, False)])
def test_int8_product_with_token_scales(model, rock, loads, shape, transB, extra, out, vector, bias):
    m, n, k = shape
    rng = np.random.default_rng(m + n + k)
    A = rng.integers(-128, 128, (m, k)).astype(np.int8)
    B = rng.integers(-128, 128, (n, k) if transB else (k, n)).astype(np.int8)
    token = rng.uniform(0.001, 0.01, m).astype(np.float32)
    channel = rng.uniform(0.01, 0.1, n).astype(np.float32)
    bv = rng.integers(-4, 5, n).astype(np.float32)
    opts = ("-operation gemm -arch gfx950 -t i8 -m %d -n %d -k %d -transB %s -out_datatype %s -token_scale_vector true -zero_point 3 %s"
            % (m, n, k, flag(transB), out, extra))
    inputs = {0: A, 1: B, 4: token}
    if vector:
        opts += " -scale_vector true"
        inputs[5] = channel
    else:
        opts += " -scale 0.03125 -activation clip -clip_min -2 -clip_max 3"
    if bias:
        opts += " -bias true"
        inputs[3] = bv
    names, problems, got = run_plan(model, rock, opts, inputs)
    assert not problems, (names, problems)
    acc = A.astype(np.int64) @ (B.T if transB else B).astype(np.int64)
    want = scaled(acc, 3, channel if vector else np.full(n, 0.03125), token, bv if bias else None, "f32")
    if not vector:
        want = np.clip(want, -2, 3)
    want = want.astype(_NUMPY[out])
    assert np.array_equal(got[2][:want.nbytes].view(want.dtype).reshape(m, n), want), names


# ---- products grouped by expert -----------------------------------------------------------------------------------
# (groups' sizes, rows behind the last group, N, K): empty groups, one row, tiles that end inside a group, 70 groups
GROUPS = [([5], 0, 24, 32), ([0, 3, 0, 64, 1, 0], 3, 40, 64), ([130, 0, 7], 5, 72, 48), ([0, 0], 4, 16, 32),
          ([1] * 70 + [0, 9], 2, 16, 32), ([17, 40], 0, 33, 35), ([3, 66, 2], 1, 77, 64), ([130, 0, 90], 2, 45, 37),
          ([200, 0, 70], 1, 5, 3), ([1, 200], 0, 9, 131)]


def _problem(sizes, tail, n, k, t, transB, seed=0):
    rng = np.random.default_rng(seed + sum(sizes))
    T = sum(sizes) + tail
    offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    E = len(sizes)
    x = rng.integers(-3, 4, (T, k)).astype(_NUMPY[t])
    w = rng.integers(-3, 4, (E, n, k) if transB else (E, k, n)).astype(_NUMPY[t])
    return rng, T, E, offsets, x, w


def _opts(op, t, T, E, n, k, transB, extra=""):
    return "-operation %s -arch gfx950 -t %s -g %d -m %d -n %d -k %d -transB %s %s" % (op, t, E, T, n, k, flag(transB), extra)


@pytest.mark.parametrize("case", GROUPS, ids=lambda c: "%dgroups-%dx%d" % (len(c[0]), c[2], c[3]))
@pytest.mark.parametrize("t,transB", [("f16", True), ("f16", False), ("f32", True), ("i8", True), ("i8", False)])
def test_grouped_product(model, rock, loads, case, t, transB):
    sizes, tail, n, k = case
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, transB)
    inputs, extra, out = {0: x, 1: w, 3: offsets}, "", t
    if t == "i8":
        token, channel = rng.uniform(0.5, 1, T).astype(np.float32), rng.uniform(0.1, 0.5, (E, n)).astype(np.float32)
        inputs.update({4: token, 5: channel})
        extra, out = "-token_scale_vector true -scale_vector true -out_datatype f32", "f32"
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", t, T, E, n, k, transB, extra), inputs)
    assert not problems, (names, problems)
    res = got[2][:T * n * np.dtype(_NUMPY[out]).itemsize].view(_NUMPY[out]).reshape(T, n)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        acc = x[a:b].astype(np.float64) @ (w[e].T if transB else w[e]).astype(np.float64)
        want = scaled(acc, 0, channel[e], token[a:b], None, "f32") if t == "i8" else acc
        assert np.array_equal(res[a:b].astype(np.float64), want.astype(np.float64)), (names, e)
    assert (res[sum(sizes):].view(np.uint8) == 0xEE).all(), "rows behind the last group were written"


@pytest.mark.parametrize("case", GROUPS, ids=lambda c: "%dgroups-%dx%d" % (len(c[0]), c[2], c[3]))
@pytest.mark.parametrize("t,transB", [("f16", True), ("f16", False), ("f32", True)])
def test_grouped_gradients(model, rock, loads, case, t, transB):
    sizes, tail, n, k = case
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, transB)
    dout = rng.integers(-3, 4, (T, n)).astype(_NUMPY[t])
    dout[sum(sizes):] = np.nan      # rows of no group: read by nothing
    x[sum(sizes):] = np.nan
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_data", t, T, E, n, k, transB),
                                    {1: w, 2: dout, 3: offsets})
    assert not problems, (names, problems)
    dx = got[0][:x.nbytes].view(x.dtype).reshape(T, k).copy()   # (the next plan reuses the memory)
    names_w, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", t, T, E, n, k, transB),
                                      {0: x, 2: dout, 3: offsets})
    assert not problems, (names_w, problems)
    dw = got[1][:w.nbytes].view(w.dtype).reshape(w.shape)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        we = (w[e] if transB else w[e].T).astype(np.float64)     # [N, K]
        d64, x64 = dout[a:b].astype(np.float64), x[a:b].astype(np.float64)
        assert np.array_equal(dx[a:b].astype(np.float64), d64 @ we), (names, e)
        want = d64.T @ x64 if transB else x64.T @ d64
        assert np.array_equal(dw[e].astype(np.float64), want), (names_w, e)
    assert (dx[sum(sizes):].view(np.uint8) == 0xEE).all()


@pytest.mark.parametrize("tile", ["v2:256,256", "v2:128,128", "v2:64,64"])
@pytest.mark.parametrize("t,transB", [("f16", True), ("f16", False), ("i8", True)])
def test_grouped_product_every_tile(model, rock, loads, tile, t, transB):
    """Groups that end inside a tile, at a tile's end and one row behind it, on every tile."""
    sizes, tail, n, k = [64, 0, 129, 257, 1], 2, 272, 80
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, transB)
    extra = "-perf_config " + tile + (" -out_datatype f32" if t == "i8" else "")
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", t, T, E, n, k, transB, extra),
                                    {0: x, 1: w, 3: offsets})
    assert not problems and tile[3:].replace(",", "x") in names[0], (names, problems)
    out = np.float32 if t == "i8" else _NUMPY[t]
    res = got[2][:T * n * np.dtype(out).itemsize].view(out).reshape(T, n)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        assert np.array_equal(res[a:b].astype(np.float64), x[a:b].astype(np.float64) @ (w[e].T if transB else w[e]).astype(np.float64)), e


@pytest.mark.parametrize("tile", ["v2:256,256", "v2:128,128", "v2:64,64"])
def test_grouped_weight_gradient_every_tile(model, rock, loads, tile):
    sizes, tail, n, k = [64, 0, 129, 1], 2, 272, 136
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, "f16", True)
    dout = rng.integers(-3, 4, (T, n)).astype(np.float16)
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", "f16", T, E, n, k, True, "-perf_config " + tile),
                                    {0: x, 2: dout, 3: offsets})
    assert not problems and tile[3:].replace(",", "x") in names[0], (names, problems)
    dw = got[1][:w.nbytes].view(w.dtype).reshape(w.shape)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        assert np.array_equal(dw[e].astype(np.float64), dout[a:b].astype(np.float64).T @ x[a:b].astype(np.float64)), e


@pytest.mark.parametrize("tile", ["v2:128,128", "v2:64,64"])
@pytest.mark.parametrize("t,transB", [("f16", True), ("f16", False), ("f32", False), ("i8", True)])
@pytest.mark.parametrize("n,k", [(150, 77), (133, 261), (9, 200)])
def test_every_tile_of_any_alignment(model, rock, loads, tile, t, transB, n, k):
    """Rows that are no whole chunks: products, gradient of the rows, gradient of the weights; ends of rows inside a
    chunk, a K-step of all zeros but one element, columns of one chunk."""
    sizes, tail = [129, 0, 70, 1], 1
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, transB)
    extra = "-perf_config " + tile + (" -out_datatype f32" if t == "i8" else "")
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", t, T, E, n, k, transB, extra), {0: x, 1: w, 3: offsets})
    es = np.dtype(_NUMPY[t]).itemsize
    chunks = lambda c: c * es % 16 == 0   # noqa: E731
    assert not problems and tile[3:].replace(",", "x") in names[0], (names, problems)
    assert ("_any" in names[0]) == (not (chunks(k) and (transB or chunks(n)))), names
    out = np.float32 if t == "i8" else _NUMPY[t]
    res = got[2][:T * n * np.dtype(out).itemsize].view(out).reshape(T, n)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        want = x[a:b].astype(np.float64) @ (w[e].T if transB else w[e]).astype(np.float64)
        assert np.array_equal(res[a:b], want.astype(out)), e
    assert (res[sum(sizes):].view(np.uint8) == 0xEE).all()
    if t == "i8":
        return
    dout = rng.integers(-3, 4, (T, n)).astype(_NUMPY[t])
    dout[sum(sizes):] = np.nan
    x[sum(sizes):] = np.nan
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", t, T, E, n, k, transB, extra),
                                    {0: x, 2: dout, 3: offsets})
    assert not problems and tile[3:].replace(",", "x") in names[0], (names, problems)
    assert ("_any" in names[0]) == (not (chunks(k) and chunks(n))), names
    dw = got[1][:w.nbytes].view(w.dtype).reshape(w.shape)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        d64, x64 = dout[a:b].astype(np.float64), x[a:b].astype(np.float64)
        assert np.array_equal(dw[e].astype(np.float64), d64.T @ x64 if transB else x64.T @ d64), e


@pytest.mark.parametrize("groups", [300, 350], ids=["quarters", "halves"])
def test_last_tiles_in_parts(model, rock, groups):
    """More 256 x 256 tiles than compute units: 256 whole ones, then 44 in quarters or 94 in halves.  Groups of one to three
    rows, each a tile of its own; the blocks from number 250 on run (the GPU tests run whole launches)."""
    sizes, n = [1 + g % 3 for g in range(groups)], 256
    rng, T, E, offsets, x, w = _problem(sizes, 1, n, 16, "f16", True)
    opts = _opts("grouped_gemm", "f16", T, E, n, 16, True, "-perf_config v2:256,256")
    model.hm_set_blocks(250, 1 << 20)
    try:
        names, problems, got = run_plan(model, rock, opts, {0: x, 1: w, 3: offsets})
    finally:
        model.hm_set_blocks(0, 0xFFFFFFFF)
    assert not problems and "256x256" in names[0], (names, problems)
    res = got[2][:T * n * 2].view(np.float16).reshape(T, n)
    done = 0
    for e, (a, b) in enumerate(bounds(offsets, T)):
        if e < 256 and (res[a:b].view(np.uint8) == 0xEE).all():
            continue   # a whole tile of a block that did not run
        done += 1
        assert np.array_equal(res[a:b].astype(np.float64), x[a:b].astype(np.float64) @ w[e].T.astype(np.float64)), e
    assert done == groups - 250
    assert (res[sum(sizes):].view(np.uint8) == 0xEE).all()


@pytest.mark.parametrize("tile", ["v2:16,16", "v2:16,32", "v2:32,16", "v2:32,32"])
@pytest.mark.parametrize("t", ["f16", "f32", "i8"])
@pytest.mark.parametrize("n,k", [(70, 35), (36, 1040), (33, 2501)])
def test_grouped_product_every_kernel_for_few_rows(model, rock, tile, t, n, k):
    """Depths below one K-step, of whole steps for every wave, and with a remainder behind them; columns that end
    inside a tile; groups larger than the tile."""
    sizes, tail = [1, 0, 17, 70, 3], 2
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, True)
    extra = "-perf_config " + tile + (" -out_datatype f32" if t == "i8" else "")
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", t, T, E, n, k, True, extra), {0: x, 1: w, 3: offsets})
    assert not problems and tile[3:].replace(",", "x") + "_skinny" in names[0], (names, problems)
    out = np.float32 if t == "i8" else _NUMPY[t]
    res = got[2][:T * n * np.dtype(out).itemsize].view(out).reshape(T, n)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        want = x[a:b].astype(np.float64) @ w[e].T.astype(np.float64)
        assert np.array_equal(res[a:b], want.astype(out)), e
    assert (res[sum(sizes):].view(np.uint8) == 0xEE).all()


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("transB", [True, False])
@pytest.mark.parametrize("sizes", [[700, 0, 33, 1], [64], [257, 512]])
def test_weight_gradient_split_over_the_waves(model, rock, loads, t, transB, sizes):
    """Shares with several K-steps, with one, with none; groups without rows."""
    tail, n, k = 2, 136, 72
    rng, T, E, offsets, x, w = _problem(sizes, tail, n, k, t, transB)
    dout = rng.integers(-3, 4, (T, n)).astype(_NUMPY[t])
    dout[sum(sizes):] = np.nan
    x[sum(sizes):] = np.nan
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", t, T, E, n, k, transB, "-perf_config v2:64,64,8,32,16,8,4,1,1"),
                                    {0: x, 2: dout, 3: offsets})
    assert not problems and names[0].endswith("_64x64_split"), (names, problems)
    dw = got[1][:w.nbytes].view(w.dtype).reshape(w.shape)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        d64, x64 = dout[a:b].astype(np.float64), x[a:b].astype(np.float64)
        assert np.array_equal(dw[e].astype(np.float64), (d64.T @ x64 if transB else x64.T @ d64).astype(_NUMPY[t])), e


@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 2, 100, 7], [4, 4, 4, 2], [9, 0, 0, 0], [2147483647] * 4, [-2147483648, 1, 1, 12]])
def test_offsets_that_are_no_offsets_stay_inside_the_tensors(model, rock, offsets):
    """Boundaries that step back or lie outside are read as the furthest one before them: nothing outside the tensors
    is touched, no row belongs to two groups."""
    T, n, k = 12, 24, 32
    rng = np.random.default_rng(5)
    x, w = rng.integers(-3, 4, (T, k)).astype(np.float16), rng.integers(-3, 4, (3, n, k)).astype(np.float16)
    dout = rng.integers(-3, 4, (T, n)).astype(np.float16)
    off = np.asarray(offsets, np.int64).astype(np.int32)
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", "f16", T, 3, n, k, True), {0: x, 1: w, 3: off})
    assert not problems, (names, problems)
    res = got[2][:T * n * 2].view(np.float16).reshape(T, n)
    owned = np.zeros(T, bool)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        assert np.array_equal(res[a:b].astype(np.float64), x[a:b].astype(np.float64) @ w[e].T.astype(np.float64))
        owned[a:b] = True
    assert (res[~owned].view(np.uint8) == 0xEE).all()
    for op, inputs in (("grouped_gemm_bwd_data", {1: w, 2: dout, 3: off}), ("grouped_gemm_bwd_weight", {0: x, 2: dout, 3: off})):
        names, problems, _ = run_plan(model, rock, _opts(op, "f16", T, 3, n, k, True), inputs)
        assert not problems, (names, problems)


# boundaries that step back right away, out of the rows, and far behind the furthest one (another lane group's)
STEPPING_BACK = [[0, 5, 3, 9], [-4, 2, 100, 7], [9, 0, 0, 0], [2147483647] * 4, [-2147483648, 1, 1, 12], [3, 2, 1, 0, 200, 150, 131],
                 [0, 40, 7] + [8] * 80 + [60, 2, 90] + [0] * 70 + [130, 5]]


@pytest.mark.parametrize("offsets", STEPPING_BACK, ids=lambda o: "-".join(map(str, o[:7])))
@pytest.mark.parametrize("n,k,perf", [(24, 32, ""), (24, 32, "v2:64,64,8,32,16,8,4,1,1"), (24, 32, "v2:128,128"), (24, 32, "v2:256,256"),
                                      (21, 33, "v2:64,64"), (21, 33, "v2:128,128")],
                         ids=["chosen", "split", "128", "256", "any64", "any128"])
def test_gradients_on_offsets_that_step_back(model, rock, offsets, n, k, perf):
    """Both gradients read the boundaries as the product does: a row counts in one group's gradient at most."""
    T, E = 131, len(offsets) - 1
    rng = np.random.default_rng(7)
    x, w = rng.integers(-3, 4, (T, k)).astype(np.float16), rng.integers(-3, 4, (E, n, k)).astype(np.float16)
    dout = rng.integers(-3, 4, (T, n)).astype(np.float16)
    off = np.asarray(offsets, np.int64).astype(np.int32)
    extra = "-perf_config " + perf if perf else ""
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", "f16", T, E, n, k, True, extra), {0: x, 2: dout, 3: off})
    assert not problems, (names, problems)
    dw = got[1][:w.nbytes].view(w.dtype).reshape(w.shape)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        assert np.array_equal(dw[e].astype(np.float64), dout[a:b].astype(np.float64).T @ x[a:b].astype(np.float64)), (names, e)
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_data", "f16", T, E, n, k, True), {1: w, 2: dout, 3: off})
    assert not problems, (names, problems)
    dx, owned = got[0][:x.nbytes].view(x.dtype).reshape(T, k), np.zeros(T, bool)
    for e, (a, b) in enumerate(bounds(offsets, T)):
        assert np.array_equal(dx[a:b].astype(np.float64), dout[a:b].astype(np.float64) @ w[e].astype(np.float64)), (names, e)
        owned[a:b] = True
    assert (dx[~owned].view(np.uint8) == 0xEE).all()


class _Sparse:
    """A tensor whose pages exist where they are touched only."""

    def __init__(self, nbytes):
        import mmap
        noreserve = 0x4000
        self.map = mmap.mmap(-1, nbytes, flags=mmap.MAP_SHARED | mmap.MAP_ANONYMOUS | noreserve)
        self.bytes = np.frombuffer(self.map, np.uint8)
        self.at = self.bytes.ctypes.data

    def of(self, dtype, shape):
        return self.bytes[:int(np.prod(shape, dtype=np.int64)) * np.dtype(dtype).itemsize].view(dtype).reshape(shape)


@pytest.mark.parametrize("depth", [1, 9], ids=["elements", "chunks"])
@pytest.mark.parametrize("op,t", [("grouped_gemm", "f16"), ("grouped_gemm", "f32"), ("grouped_gemm_bwd_weight", "f16")])
def test_rows_longer_than_two_gibibytes(model, rock, op, t, depth):
    """Columns whose byte position in their row passes 2^31, in K-major operands of any alignment: the last two tiles of a
    launch, on tensors that are mostly holes."""
    weight, ty = op != "grouped_gemm", _NUMPY[t]
    es = np.dtype(ty).itemsize
    wide, rows = (1 << 31) // es + 203, 9 if weight else 2
    # product: x [rows, depth] times w [depth, wide]; weight gradient: x [depth, wide], dout [depth, rows] -> [wide, rows]
    opts = _opts(op, t, *((depth, 1, rows, wide) if weight else (rows, 1, wide, depth)), False, "-perf_config v2:128,128")
    k = rock.RockKernel(opts)
    assert "_128x128_any" in k.kernel_name and k.block_size == 256
    tensors = [_Sparse(int(np.prod(dims, dtype=np.int64)) * 4 + 4096) for _, dims in k.arguments()]
    rng = np.random.default_rng(depth)
    small = rng.integers(-3, 4, (depth, rows) if weight else (rows, depth)).astype(ty)
    wide_tensor = tensors[0 if weight else 1].of(ty, (depth, wide))
    tail = 75 + 128                                            # columns of the last two tiles
    wide_tensor[:, -tail - 40:] = rng.integers(-3, 4, (depth, tail + 40))
    tensors[2 if weight else 0].of(ty, small.shape)[:] = small
    tensors[3].of(np.int32, (2,))[:] = [0, depth if weight else rows]
    ptrs = (C.c_void_p * 8)()
    for j, (src, off) in enumerate(pointer_map(rock, k)):
        ptrs[j] = None if src < 0 else tensors[src].at + off
    text = C.create_string_buffer(512)
    model.hm_clear()
    model.hm_set_blocks(k.grid_size - 2, 2)
    try:
        bad = model.hm_run(k.kernel_name.encode(), k.params(), ptrs, k.grid_size, k.block_size, text, 512)
    finally:
        model.hm_set_blocks(0, 0xFFFFFFFF)
    assert bad == 0, text.value
    columns = wide_tensor[:, -tail:].astype(np.float64)
    if weight:
        got, want = tensors[1].of(ty, (wide, rows))[-tail:], columns.T @ small.astype(np.float64)
    else:
        got, want = tensors[2].of(ty, (rows, wide))[:, -tail:], small.astype(np.float64) @ columns
    assert np.array_equal(got.astype(np.float64), want)


def test_offsets_beyond_the_rows_are_clamped(model, rock):
    """As the header and grouped_gemm() say: below 0 is 0, beyond the rows is their number, stepping back is the furthest
    one before.  [-4, 2, 100, 7] over 12 rows: group 0 has the rows 0 and 1, group 1 the rest, group 2 none."""
    T, n, k = 12, 24, 32
    x, w = np.ones((T, k), np.float16), np.stack([np.full((n, k), v, np.float16) for v in (1, 2, 3)])
    off = np.array([-4, 2, 100, 7], np.int32)
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm", "f16", T, 3, n, k, True), {0: x, 1: w, 3: off})
    assert not problems, (names, problems)
    res = got[2][:T * n * 2].view(np.float16).reshape(T, n)
    assert (res[:2] == k).all() and (res[2:] == 2 * k).all()
    names, problems, got = run_plan(model, rock, _opts("grouped_gemm_bwd_weight", "f16", T, 3, n, k, True),
                                    {0: x, 2: np.ones((T, n), np.float16), 3: off})
    assert not problems, (names, problems)
    dw = got[1][:w.nbytes].view(np.float16).reshape(w.shape)
    assert (dw[0] == 2).all() and (dw[1] == 10).all() and (dw[2] == 0).all()
