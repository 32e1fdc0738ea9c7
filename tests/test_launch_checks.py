"""What rockamdLaunch refuses before it touches the device: tensors that a kernel of the list reads or writes and that
the caller left out.  Addresses here are numbers that nothing reads: a launch that passes the checks ends at the
missing device, so these tests run where there is none."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a launch that passes the checks would run on the device")

ATTENTION = "-operation attention -arch gfx950 -t f16 -g 1 -seq_len_q 64 -seq_len_k 64 "


def refused(rock, options, missing):
    """Whether the launch check refuses the kernel without the tensors `missing` (positions in the caller's list)."""
    lib = rock.load_library()
    k = rock.RockKernel(options)
    pointers = (C.c_void_p * k.caller_pointers)(*[None if i in missing else 0x100000 * (i + 1) for i in range(k.caller_pointers)])
    assert lib.rockamdLaunch(k._h, pointers, k.caller_pointers, None) != 0
    return "NULL tensor pointer" in rock.api.last_error(), k


@pytest.mark.parametrize("inputs", [1, 2, 3])
def test_the_row_softmax_needs_the_tensors_of_its_program(rock, inputs):
    """They stand between V and O in the caller's list -- the first where other problems have the optional bias -- and
    reach the kernel through its parameter block."""
    program = "x" + "".join(",t%d,add" % i for i in range(inputs))
    options = ATTENTION + "-head_dim_qk 32 -head_dim_v 32 -attn_elementwise %s -attn_inputs %s -kernel_id 1" % (program, ",".join(["f16"] * inputs))
    for i in range(inputs):
        no, k = refused(rock, options, {3 + i})
        assert k.kernel_name == "rock_softmax_rows" and k.caller_pointers == 5 + inputs
        assert no, "launched without t%d" % i
    assert refused(rock, options, {4 + inputs})[0]                 # the workspace with the scores
    assert not refused(rock, options, {0, 1, 2, 3 + inputs})[0]    # Q, K, V and O are the products'
    assert not refused(rock, options, set())[0]


def test_the_row_softmax_needs_its_own_scale_tensor_and_bias(rock):
    options = ATTENTION + "-head_dim_qk 300 -head_dim_v 300 -with-attn-scale true -with-attn-bias true -kernel_id 1"
    for i, needed in enumerate([False, False, False, True, True, False, True]):     # Q, K, V, scale, bias, O, workspace
        no, k = refused(rock, options, {i})
        assert k.kernel_name == "rock_softmax_rows" and k.caller_pointers == 7
        assert no == needed, i


def test_a_copy_needs_its_two_tensors_only(rock):
    """Padded copies around the fused kernel: the bias slot, which is not where it is without a scale tensor, may be
    empty."""
    options = ATTENTION + "-head_dim_qk 36 -head_dim_v 36 -with-attn-scale true "
    no, first = refused(rock, options, {4})
    assert first.kernel_name.startswith("rock_relayout") and not no
    for i, needed in enumerate([True, False, False, False, False, False, True]):    # Q, K, V, scale, bias slot, O, workspace
        assert refused(rock, options, {i})[0] == needed, i


def test_a_bias_slot_stays_optional(rock):
    gemm = "-operation gemm -arch gfx950 -t f16 -m 64 -n 64 -k 64"
    assert not refused(rock, gemm, {3})[0] and refused(rock, gemm + " -bias true", {3})[0]
    for i in range(3):
        assert refused(rock, gemm, {i})[0]
    grouped = "-operation grouped_gemm -arch gfx950 -t f16 -g 2 -m 64 -n 64 -k 64"
    for i in range(4):
        assert refused(rock, grouped, {i})[0]
