"""What the operators over token rows refuse, on the host, before anything is launched: through the package's entry points
(with tensors on the CPU, which get no further than the checks) and through option strings."""
import pytest
import torch


def _t(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


OFF3 = torch.zeros(4, dtype=torch.int32)
I8 = torch.int8


@pytest.mark.parametrize("call,text", [
    (lambda r: r.quantize_tokens(_t(4, 8, dtype=torch.int8)), "f16, bf16 or f32"),
    (lambda r: r.quantize_tokens(torch.tensor(1.0)), "f16, bf16 or f32"),
    (lambda r: r.quantize_tokens(_t(4, 8), out=_t(4, 8)), "out must be"),
    (lambda r: r.quantize_tokens(_t(4, 8), out=_t(8, 4, dtype=I8).t()), "contiguous"),
    (lambda r: r.quantize_tokens(_t(4, 8), scale_out=_t(4)), "out must be"),
    (lambda r: r.gemm(_t(4, 8), _t(6, 8), transB=True, token_scale=torch.ones(4)), "int8 operands"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(6)), "token_scale must hold 4"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4).half()), "token_scale must hold"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4), scale=torch.ones(4)), "scale must hold 6"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4), bias=torch.ones(4)), "bias must hold 6"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 9, dtype=I8), transB=True, token_scale=torch.ones(4)), "shapes do not match"),
    (lambda r: r.gemm(_t(2, 4, 8, dtype=I8), _t(2, 6, 8, dtype=I8), transB=True, token_scale=torch.ones(4)), "one batch entry"),
    (lambda r: r.gemm(_t(8, 4, dtype=I8), _t(6, 8, dtype=I8), transA=True, transB=True, token_scale=torch.ones(4)), "takes scale"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4), residual=_t(4, 6)), "takes scale"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4), out_dtype="i32"), "out_dtype"),
    (lambda r: r.gemm(_t(4, 8, dtype=I8), _t(6, 8, dtype=I8), transB=True, token_scale=torch.ones(4), activation="gelu"), "relu and clip"),
    (lambda r: r.gemm(_t(1, 131072, dtype=I8), _t(1, 131072, dtype=I8), transB=True, token_scale=torch.ones(1)), "131071"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3.long(), transB=True), "offsets is int32"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3[:3], transB=True), "offsets is int32"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(0, 6, 8), OFF3[:1], transB=True), "no experts"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3), "shapes do not match"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8, dtype=torch.bfloat16), OFF3, transB=True), "of one type"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3, transB=True, scale=2.0), "scales go with int8"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3, transB=True, token_scale=torch.ones(5)), "scales go with int8"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3, transB=True, out_dtype="i8"), "out_dtype"),
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3, transB=True, out=_t(5, 8)), "out must be"),
    (lambda r: r.grouped_gemm(_t(5, 8, dtype=I8), _t(3, 6, 8, dtype=I8), OFF3, transB=True, scale=torch.ones(6)), "scale must hold 18"),
    (lambda r: r.grouped_gemm(_t(5, 8, dtype=torch.float64), _t(3, 6, 8, dtype=torch.float64), OFF3, transB=True), "unsupported tensor dtype"),
    (lambda r: r.grouped_gemm_bwd_data(_t(5, 8), _t(3, 6, 8), OFF3, transB=True), "shapes do not match"),
    (lambda r: r.grouped_gemm_bwd_data(_t(5, 6, dtype=I8), _t(3, 6, 8, dtype=I8), OFF3, transB=True), "f16, bf16 or f32"),
    (lambda r: r.grouped_gemm_bwd_weight(_t(5, 8), _t(4, 6), OFF3), "of one type"),
    (lambda r: r.grouped_gemm_bwd_weight(_t(5, 8), _t(5, 6), OFF3, out=_t(3, 6, 8)), "out must be"),
    (lambda r: r.grouped_gemm_bwd_weight(_t(5, 8), _t(5, 6), OFF3.float()), "offsets is int32"),
    (lambda r: (lambda x: r.grouped_gemm(x, _t(1, 8, 8), OFF3[:2], transB=True, out=x))(_t(5, 8)), "overlaps an operand"),
    (lambda r: (lambda b: r.grouped_gemm(b[:5], _t(1, 8, 8), OFF3[:2], transB=True, out=b[4:9]))(_t(9, 8)), "overlaps an operand"),
    (lambda r: (lambda b: r.grouped_gemm_bwd_weight(_t(5, 8), b[0, :5], OFF3[:2], out=b[:, :8]))(_t(1, 16, 6)), "overlaps an operand"),
    # tensors that pass every check but do not live on a GPU
    (lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), OFF3, transB=True), "must live on the GPU"),
    (lambda r: r.quantize_tokens(_t(5, 8)), "must live on the GPU"),
], ids=lambda v: v.replace(" ", "-") if isinstance(v, str) else "")
def test_entry_points_refuse(rock, call, text):
    with pytest.raises(rock.RockError, match=text):
        call(rock)


@pytest.mark.parametrize("options,text", [
    ("-operation quantize_tokens -t i8 -m 4 -k 4", "quantize_tokens"),
    ("-operation quantize_tokens -t f16 -m 0 -k 4", "positive"),
    ("-operation quantize_tokens -t f16 -m 4", "positive"),
    ("-operation quantize_tokens -t f16 -m 4 -k 4 -kernel_id 1", "kernel_id"),
    ("-operation grouped_gemm -t fp8 -g 2 -m 4 -n 8 -k 16", "operands are"),
    ("-operation grouped_gemm -t f16 -g 0 -m 4 -n 8 -k 16", "positive"),
    ("-operation grouped_gemm -t f16 -g 2 -m 4 -n 8", "positive"),
    ("-operation grouped_gemm -t f16 -g 65537 -m 4 -n 8 -k 16", "at most 65536"),
    ("-operation grouped_gemm -t f16 -g 2 -m 4 -n 8 -k 16 -transA true", "no transA"),
    ("-operation grouped_gemm -t f16 -g 2 -m 4 -n 8 -k 16 -bias true", "no bias"),
    ("-operation grouped_gemm -t f16 -g 2 -m 4 -n 8 -k 16 -token_scale_vector true", "scales go with int8"),
    ("-operation grouped_gemm -t f16 -g 2 -m 4 -n 8 -k 16 -out_datatype i8", "the result is"),
    ("-operation grouped_gemm -t f16 -g 2 -m 2147483000 -n 2147483000 -k 16", "more tiles"),
    ("-operation grouped_gemm_bwd_weight -t i8 -g 2 -m 4 -n 8 -k 16", "gradients take"),
    ("-operation grouped_gemm_bwd_data -t f16 -g 2 -m 4 -n 8 -k 16 -out_datatype f32", "its tensor's type"),
    ("-operation gemm -t i8 -g 2 -m 4 -n 8 -k 16 -token_scale_vector true", "one batch entry"),
    ("-operation gemm -t f16 -m 4 -n 8 -k 16 -token_scale_vector true", "int8 operands"),
    ("-operation gemm -t i8 -m 4 -n 8 -k 16 -token_scale_vector true -activation tanh", "relu and clip"),
    ("-operation gemm -t i8 -m 4 -n 8 -k 16 -token_scale_vector true -residual add", "no residual"),
    ("-operation gemm -t i8 -m 4 -n 8 -k 16 -token_scale_vector true -store-method atomic_add", "token scales"),
    ("-operation conv -t i8 -token_scale_vector true", "gemm and grouped_gemm only"),
])
def test_option_strings_refuse(rock, options, text):
    with pytest.raises(rock.RockError, match=text):
        rock.RockKernel(options)


def test_argument_sizes_are_checked(rock):
    """rockamdCheckArgumentSizes knows every tensor of the new operators."""
    import ctypes as C
    k = rock.RockKernel("-operation grouped_gemm -t i8 -g 3 -m 5 -n 8 -k 16 -transB true -token_scale_vector true -scale_vector true")
    need = [5 * 16, 3 * 8 * 16, 5 * 8 * 2, 4 * 4, 5 * 4, 3 * 8 * 4]
    lib = rock.load_library()
    assert lib.rockamdCheckArgumentSizes(k._h, (C.c_size_t * 6)(*need), 6) == 0
    for i in range(6):
        short = list(need)
        short[i] -= 1
        assert lib.rockamdCheckArgumentSizes(k._h, (C.c_size_t * 6)(*short), 6) != 0, i


def test_tuning_space_of_the_new_operators(rock):
    k = rock.RockKernel("-operation grouped_gemm -t f16 -g 3 -m 500 -n 256 -k 64 -transB true")
    space = k.tuning_space()
    assert len(space) >= 3
    for perf in space:
        assert rock.RockKernel(k.options + " -perf_config " + perf).perf_config == perf
    assert len(rock.RockKernel("-operation quantize_tokens -t f16 -m 5 -k 8").tuning_space()) == 1


def _i8_gemm(r, **kw):
    return r.gemm(_t(4, 16, dtype=I8), _t(4, 16, dtype=I8), transB=True, out_dtype="f32", **dict(dict(token_scale=torch.ones(4)), **kw))


def _i8_grouped(r, **kw):
    return r.grouped_gemm(_t(4, 16, dtype=I8), _t(1, 4, 16, dtype=I8), OFF3[:2], transB=True, out_dtype="f32", **kw)


@pytest.mark.parametrize("call", [
    lambda r, b: _i8_gemm(r, out=b[:16].view(4, 4), token_scale=b[12:16]),
    lambda r, b: _i8_gemm(r, out=b[:16].view(4, 4), scale=b[4:8]),
    lambda r, b: _i8_gemm(r, out=b[:16].view(4, 4), bias=b[:4]),
    lambda r, b: _i8_grouped(r, out=b[:16].view(4, 4), token_scale=b[12:16]),
    lambda r, b: _i8_grouped(r, out=b[:16].view(4, 4), scale=b[4:8].view(1, 4)),
    lambda r, b: _i8_grouped(r, out=b[:16].view(4, 4), token_scale=b[13:30:5]),       # (copied first, refused all the same)
    lambda r, b: r.quantize_tokens(_t(4, 16), out=b.view(I8)[:64].view(4, 16), scale_out=b[12:16]),
    lambda r, b: r.quantize_tokens(b[:16].view(4, 4), scale_out=b[12:16]),
])
def test_results_may_not_overlap_scales_or_each_other(rock, call):
    with pytest.raises(rock.RockError, match="overlaps"):
        call(rock, torch.zeros(64))


def test_results_beside_scales_are_taken(rock):
    """The same tensors without the overlap get as far as the device check."""
    b = torch.zeros(64)
    for call in (lambda: _i8_gemm(rock, out=b[:16].view(4, 4), token_scale=b[16:20], scale=b[20:24], bias=b[24:28]),
                 lambda: _i8_grouped(rock, out=b[:16].view(4, 4), token_scale=b[16:20], scale=b[20:24].view(1, 4)),
                 lambda: rock.quantize_tokens(b[32:].view(4, 8), out=b.view(I8)[:32].view(4, 8), scale_out=b[8:12])):
        with pytest.raises(rock.RockError, match="must live on the GPU"):
            call()


def test_an_empty_dimension_of_the_result_is_an_empty_result(rock):
    """Nothing to compute: the (empty) result, checked like any other."""
    e8 = torch.zeros((0, 16), dtype=I8)
    assert rock.gemm(_t(4, 16, dtype=I8), e8, transB=True, token_scale=torch.ones(4)).shape == (4, 0)
    assert rock.gemm(_t(4, 16, dtype=I8), e8.t(), token_scale=torch.ones(4), out_dtype="f32").dtype == torch.float32
    assert rock.gemm(e8, _t(6, 16, dtype=I8), transB=True, token_scale=torch.ones(0), bias=torch.ones(6)).shape == (0, 6)
    assert rock.grouped_gemm(_t(5, 8), _t(3, 0, 8), OFF3, transB=True).shape == (5, 0)
    assert rock.grouped_gemm(_t(5, 0), _t(3, 0, 0), OFF3).shape == (5, 0)
    assert rock.grouped_gemm(_t(0, 0), _t(3, 0, 6), OFF3).shape == (0, 6)
    assert rock.grouped_gemm_bwd_data(_t(5, 6), _t(3, 6, 0), OFF3, transB=True).shape == (5, 0)
    assert rock.grouped_gemm_bwd_data(_t(0, 0), _t(3, 0, 8), OFF3, transB=True).shape == (0, 8)
    assert rock.grouped_gemm_bwd_weight(_t(5, 0), _t(5, 6), OFF3).shape == (3, 0, 6)
    with pytest.raises(rock.RockError, match="token_scale must hold 4"):
        rock.gemm(_t(4, 16, dtype=I8), e8, transB=True, token_scale=torch.ones(3))
    with pytest.raises(rock.RockError, match="out must be"):
        rock.grouped_gemm(_t(5, 8), _t(3, 0, 8), OFF3, transB=True, out=_t(5, 1))


@pytest.mark.parametrize("call", [
    lambda r: r.gemm(_t(4, 0, dtype=I8), _t(6, 0, dtype=I8), transB=True, token_scale=torch.ones(4)),
    lambda r: r.gemm(_t(4, 0, dtype=I8), _t(0, 6, dtype=I8), token_scale=torch.ones(4)),
    lambda r: r.grouped_gemm(_t(5, 0), _t(3, 6, 0), OFF3, transB=True),
    lambda r: r.grouped_gemm(_t(5, 0, dtype=I8), _t(3, 0, 6, dtype=I8), OFF3),
    lambda r: r.grouped_gemm_bwd_data(_t(5, 0), _t(3, 0, 8), OFF3, transB=True),
    lambda r: r.grouped_gemm_bwd_data(_t(5, 0), _t(3, 8, 0), OFF3),
])
def test_an_empty_reduction_is_a_product(rock, call):
    """Not refused for its depth: it gets as far as the device check."""
    with pytest.raises(rock.RockError, match="must live on the GPU"):
        call(rock)


@pytest.mark.parametrize("shape,taken", [((3, 6), True), ((3, 1, 6), True), ((3, 6, 1), True), ((18,), True), ((6, 3), False), ((2, 9), False),
                                         ((3, 2, 3), False), ((1, 6, 3), False)])
def test_channel_scales_of_experts_in_another_order(rock, shape, taken):
    """[E, N], with dimensions of one anywhere, or flat; as many values in another order are not what the caller means."""
    with pytest.raises(rock.RockError, match="must live on the GPU" if taken else "scale is .E, N."):
        rock.grouped_gemm(_t(5, 16, dtype=I8), _t(3, 6, 16, dtype=I8), OFF3, transB=True, scale=torch.ones(shape))


@pytest.mark.parametrize("call", [
    lambda r: _i8_gemm(r, token_scale=0.5),
    lambda r: _i8_gemm(r, bias=[1.0] * 4),
    lambda r: _i8_grouped(r, token_scale=[1.0] * 4),
    lambda r: r.grouped_gemm(_t(5, 8), _t(3, 6, 8), [0, 1, 2, 3], transB=True),
    lambda r: r.grouped_gemm_bwd_data(_t(5, 6), _t(3, 6, 8), (0, 1, 2, 3), transB=True),
    lambda r: r.grouped_gemm_bwd_weight(_t(5, 8), _t(5, 6), [0, 1, 2, 3]),
])
def test_what_must_be_a_tensor(rock, call):
    with pytest.raises(rock.RockError, match="tensor|offsets is int32"):
        call(rock)


def test_a_refused_stream_leaves_the_current_device(rock, monkeypatch):
    """Whatever goes wrong with the stream of a call, the device that the call made the current one is put back."""
    import rocmlir_amd.api as api
    if api.torch is None:
        api._load_torch()
    entered = []

    class Device:
        def __init__(self, device):
            pass

        def __enter__(self):
            entered.append(1)

        def __exit__(self, *what):
            entered.append(-1)
    monkeypatch.setattr(torch.cuda, "device", Device)
    for bad in ("a stream", object()):
        with pytest.raises((rock.RockError, TypeError, ValueError)):
            api._on("test", torch.device("cuda", 0), bad)
    assert entered == [1, -1, 1, -1]
