"""The layer calls' argument checks and kernel plans (include/hexir_b200/
layers.h) without a GPU: every refusal comes before a device is opened."""

import ctypes as C

import pytest

import hexir_b200 as hx
from hexir_b200 import _ffi

P = 4096  # an aligned address that no refused call reads


def status(call, *args, **kw):
    with pytest.raises(_ffi.HexirError) as err:
        call(*args, **kw)
    return err.value.status


def linear(m=4, n=8, k=16, dtype="bf16", act="none", x=P, w=P, y=P, **kw):
    return status(hx.cuda_linear, 0, x, w, y, m, n, k, dtype, act, **kw)


BAD = _ffi.ERROR_INVALID_ARGUMENT


def test_linear_refusals():
    assert linear(dtype="f64") == _ffi.ERROR_UNIMPLEMENTED
    assert linear(dtype="f32") == _ffi.ERROR_UNIMPLEMENTED
    for ptr in ("x", "w", "y"):
        assert linear(**{ptr: 0}) == BAD
        assert linear(**{ptr: P + 1}) == BAD          # not on its elements
    for ptr in ("bias", "residual", "preact"):
        assert linear(**{ptr: P + 1}) == BAD
    assert linear(ldx=15) == BAD                        # a stride below its row
    assert linear(ldw=7) == BAD
    assert linear(ldy=7) == BAD
    assert linear(residual=P, ldr=7) == BAD
    assert linear(preact=P, ldp=7) == BAD
    assert linear(m=1 << 20, ldx=1 << 62) == BAD        # offsets past 63 bits
    assert linear(flags=0x1) == BAD
    assert linear(flags=_ffi.LINEAR_FORCE_PAIR | _ffi.LINEAR_FORCE_SINGLE) == BAD
    assert linear(flags=_ffi.LINEAR_SPLIT(3)) == BAD
    assert linear(flags=1 << 24) == BAD                 # no tile of 16 columns
    assert linear(flags=_ffi.LINEAR_FORCE_SINGLE | _ffi.LINEAR_TILE(256)) == BAD
    assert linear(m=0xFFFFFFFF) == BAD
    with pytest.raises(ValueError):
        hx.cuda_linear(0, P, P, P, 4, 8, 16, "bf16", "softmax")
    with pytest.raises(ValueError):
        hx.cuda_linear(0, P, P, P, 4, 8, 16, "int8")


def raw(fn, call):
    return getattr(hx.lib(), fn)(0, C.byref(call) if call is not None else None, None)


def test_raw_calls_refuse_null_and_unknown_codes():
    for fn in ("hexir_cuda_linear", "hexir_cuda_linear_output_grad",
               "hexir_cuda_linear_input_grad", "hexir_cuda_linear_weight_grad",
               "hexir_cuda_layer_norm", "hexir_cuda_layer_norm_grad"):
        assert raw(fn, None) == BAD
    for activation in (1, 2, 4, 11, 15, 99):            # 11: softmax, a row op
        call = _ffi.LinearCall(2, activation, 4, 8, 16, 0, P, P, 0, 0, 0, P)
        assert raw("hexir_cuda_linear", call) == BAD
    assert raw("hexir_cuda_linear", _ffi.LinearCall(4, 0, 4, 8, 16, 0, P, P, 0, 0, 0,
                                                    P)) == BAD
    call = _ffi.LinearWeightGradCall(2, 1, 4, 8, 16, 0, P, P, P)
    assert raw("hexir_cuda_linear_weight_grad", call) == BAD   # reserved
    call = _ffi.LayerNormCall(7, 8, 1, 1e-5, P, 0, 0, P)
    assert raw("hexir_cuda_layer_norm", call) == BAD


def test_grad_refusals():
    def dx(act="none", **kw):
        args = {"dz": P, "w": P, "dx": P, **{a: kw.pop(a) for a in ("dz", "w", "dx")
                                             if a in kw}}
        return status(hx.cuda_linear_input_grad, 0, args["dz"], args["w"], args["dx"],
                      4, 8, 16, "bf16", act, **kw)
    assert dx(dz=0) == dx(w=0) == dx(dx=0) == BAD
    assert dx(act="gelu") == BAD                        # no preactivations
    assert dx(lddz=7) == dx(ldw=7) == dx(lddx=15) == BAD
    assert dx(dz=P + 1) == BAD
    assert status(hx.cuda_linear_weight_grad, 0, 0, P, P, 4, 8, 16) == BAD
    assert status(hx.cuda_linear_weight_grad, 0, P, P, P, 4, 8, 16, lddw=7) == BAD
    assert status(hx.cuda_linear_weight_grad, 0, P, P, P, 4, 8, 16, "f32") == \
        _ffi.ERROR_UNIMPLEMENTED

    def out(act="none", dy=P, **kw):
        return status(hx.cuda_linear_output_grad, 0, dy, 4, 8, "bf16", act, **kw)
    assert out(dy=0, dz=P) == BAD
    assert out(act="gelu", dz=P) == BAD                 # no preactivations
    assert out(act="gelu", preact=P) == BAD             # nowhere for dz
    need = hx.grad_workspace_bytes(8, "bf16")
    assert out(dbias=P) == BAD                          # no workspace
    assert out(dbias=P, workspace=P, workspace_bytes=need - 1) == BAD
    assert out(dbias=P, workspace=P + 8, workspace_bytes=need) == BAD
    assert out(dbias=P + 1, workspace=P, workspace_bytes=need) == BAD


def test_layer_norm_refusals():
    def norm(x=P, y=P, rows=4, cols=8, dtype="f32", **kw):
        return status(hx.cuda_layer_norm, 0, x, y, rows, cols, dtype, **kw)
    assert norm(x=0) == norm(y=0) == norm(cols=0) == BAD
    assert norm(x=P + 2) == norm(gamma=P + 2) == norm(beta=P + 2) == BAD
    assert norm(mean=P + 2) == norm(rstd=P + 2) == BAD
    assert norm(ldx=7) == norm(ldy=7) == BAD
    for eps in (-1e-5, float("nan"), float("inf")):
        assert norm(eps=eps) == BAD

    def grad(dy=P, x=P, mean=P, rstd=P, dx=P, rows=4, cols=8, dtype="f64", **kw):
        return status(hx.cuda_layer_norm_grad, 0, dy, x, mean, rstd, dx, rows, cols,
                      dtype, **kw)
    assert grad(dy=0) == grad(x=0) == grad(mean=0) == grad(rstd=0) == BAD
    assert grad(cols=0) == grad(lddy=7) == grad(lddx=7) == BAD
    assert grad(residual=P, ldr=7) == grad(residual=P + 4) == BAD
    need = hx.grad_workspace_bytes(8, "f64")
    assert need == 640 * 8 * 8
    assert grad(dgamma=P) == BAD
    assert grad(dbeta=P, workspace=P, workspace_bytes=need - 1) == BAD
    assert grad(dbeta=P, workspace=P + 8, workspace_bytes=need) == BAD


@pytest.mark.skipif(hx.device_count() > 0, reason="checks the no-GPU behaviour")
def test_good_arguments_need_a_gpu():
    dev = _ffi.ERROR_DEVICE
    assert linear() == dev
    assert linear(m=0) == dev
    assert status(hx.cuda_layer_norm, 0, P, P, 4, 8) == dev
    assert status(hx.cuda_linear_weight_grad, 0, P, P, P, 4, 8, 16) == dev


def test_plans():
    PAIR, SINGLE, SKINNY, GUARDED = 1, 2, 3, 4
    assert hx.linear_plan("forward", 8192, 8192, 8192)[:2] == (PAIR, 256)
    assert hx.linear_plan("weight_grad", 8192, 8192, 8192)[:2] == (PAIR, 256)
    for m in (1, 16, 64):
        assert hx.linear_plan("forward", m, 8192, 8192)[0] == SKINNY
    assert hx.linear_plan("forward", 65, 8192, 8192)[0] != SKINNY
    assert hx.linear_plan("input_grad", 1, 8192, 8192)[0] != SKINNY
    # Few tiles and a long sum: the sum is split.
    assert hx.linear_plan("forward", 256, 512, 8192)[2] > 1
    assert hx.linear_plan("forward", 1, 8192, 8192)[2] > 1
    # No rows to load, or rows off 16 bytes.
    assert hx.linear_plan("forward", 256, 512, 0)[0] == GUARDED
    assert hx.linear_plan("forward", 256, 512, 512, aligned=False)[0] == GUARDED
    for op in ("forward", "input_grad", "weight_grad"):
        for flags, variant in ((_ffi.LINEAR_FORCE_PAIR, PAIR),
                               (_ffi.LINEAR_FORCE_SINGLE, SINGLE),
                               (_ffi.LINEAR_FORCE_GUARDED, GUARDED)):
            assert hx.linear_plan(op, 200, 264, 520, flags=flags)[0] == variant
    with pytest.raises(_ffi.HexirError):
        hx.linear_plan("forward", 65, 8, 8, flags=_ffi.LINEAR_FORCE_SKINNY)
    with pytest.raises(_ffi.HexirError):
        hx.linear_plan("input_grad", 5, 8, 8, flags=_ffi.LINEAR_FORCE_SKINNY)
    with pytest.raises(_ffi.HexirError):
        hx.linear_plan("forward", 5, 8, 8, aligned=False,
                       flags=_ffi.LINEAR_FORCE_PAIR)


def test_the_reference_slopes_are_the_activations_derivatives():
    """The formulas the GPU tests use, against central differences in 64 bits
    (off by the step's square, 1e-10, times a third derivative below 3, and by
    rounding, 1e-16 / 1e-5); corners, where the slope jumps, left out."""
    import numpy as np
    from tests import layers_reference as ref
    z = np.linspace(-9, 9, 2001)
    z = z[np.abs(z) > 1e-4]
    h = 1e-5
    for name in ref.ACTS:
        diff = (ref.act(name, z + h) - ref.act(name, z - h)) / (2 * h)
        assert np.abs(diff - ref.slope(name, z)).max() < 1e-9, name


def test_counts_beyond_32_bits_are_refused_in_python():
    """The calls' fields would cut them off without a word."""
    for bad in (1 << 32, (1 << 32) + 5, -1):
        for call in (lambda: hx.cuda_linear(0, 16, 16, 16, bad, 8, 8),
                     lambda: hx.cuda_linear(0, 16, 16, 16, 8, 8, bad),
                     lambda: hx.cuda_linear(0, 16, 16, 16, 8, 8, 8, flags=bad),
                     lambda: hx.cuda_linear_output_grad(0, 16, bad, 8),
                     lambda: hx.cuda_linear_input_grad(0, 16, 16, 16, 8, bad, 8),
                     lambda: hx.cuda_linear_weight_grad(0, 16, 16, 16, 8, 8, bad),
                     lambda: hx.cuda_layer_norm(0, 16, 16, 8, bad),
                     lambda: hx.cuda_layer_norm_grad(0, 16, 16, 16, 16, 16, 8, bad)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        hx.cuda_layer_norm(0, 16, 16, -1, 8)


def host_program(name, where):
    """A C++ test program that includes the kernels' own headers, built for
    this host."""
    import os
    import shutil
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no C++ compiler")
    exe = str(where / name)
    subprocess.run([cc, "-O1", "-std=c++17", "-Wall", "-o", exe,
                    "-I", os.path.join(here, "..", "hexir_b200", "csrc"),
                    os.path.join(here, name + ".cc")], check=True)
    return subprocess.run([exe], check=True, capture_output=True,
                          text=True).stdout.split()


def test_every_place_of_the_norm_gradients_ring_is_one_threads(tmp_path):
    """No barrier orders one thread's use of the ring against another's, so no
    place may be two threads'; zeroed as packs, a ring of single elements has
    places of other threads almost everywhere."""
    bad, mixed4, mixed2 = map(int, host_program("norm_places", tmp_path)[:3])
    assert bad == 0
    assert mixed4 > 4000 and mixed2 > 1200   # of 4096 and of 1536 elements


def test_rows_whose_blocks_reach_outside_their_tensor_are_edges(tmp_path):
    """Every offset, row length, stride and count around a pack's: rows shorter
    than a pack share the tensor's first and last block among several; of
    longer ones only the first and the last row are edges."""
    reach, needless = map(int, host_program("norm_places", tmp_path)[3:])
    assert reach == 0 and needless == 0


def test_plans_follow_the_epilogue_and_what_is_aligned():
    """What an epilogue reads, and outputs off 16 bytes, cost it more and leave
    other kernels the cheapest; the plan is told of both."""
    PAIR, SINGLE, GUARDED = 1, 2, 4
    assert hx.linear_plan("forward", 136, 5960, 8)[0] == SINGLE
    assert hx.linear_plan("forward", 136, 5960, 8, plain=True)[0] == PAIR
    assert hx.linear_plan("input_grad", 280, 8, 3416)[0] == SINGLE
    assert hx.linear_plan("input_grad", 280, 8, 3416, plain=True)[0] == PAIR
    operands = _ffi.LINEAR_ALIGNED_FIRST | _ffi.LINEAR_ALIGNED_SECOND
    assert hx.linear_plan("weight_grad", 8, 4832, 144) == \
        hx.linear_plan("weight_grad", 8, 4832, 144, plain=True) == \
        hx.linear_plan("weight_grad", 8, 4832, 144,
                       operands | _ffi.LINEAR_ALIGNED_REST)
    assert hx.linear_plan("weight_grad", 8, 4832, 144)[0] == PAIR
    assert hx.linear_plan("weight_grad", 8, 4832, 144, operands)[0] == SINGLE
    for part in (_ffi.LINEAR_ALIGNED_FIRST, _ffi.LINEAR_ALIGNED_SECOND):
        assert hx.linear_plan("forward", 256, 512, 512,
                              part | _ffi.LINEAR_ALIGNED_REST)[0] == GUARDED
    for op, empty in (("forward", (0, 8, 8)), ("forward", (8, 0, 8)),
                      ("input_grad", (8, 8, 0)), ("weight_grad", (8, 8, 0))):
        assert hx.linear_plan(op, *empty) == (0, 0, 0)
    assert hx.linear_plan("weight_grad", 0, 8, 8)[0] == GUARDED
    for bad in (dict(aligned=16), dict(flags=2), dict(flags=0x1000)):
        with pytest.raises(_ffi.HexirError):
            hx.linear_plan("forward", 8, 8, 8, **bad)
    with pytest.raises(_ffi.HexirError):
        hx.linear_plan("forward", 2 ** 31, 8, 8)       # as the call itself refuses
    assert linear(flags=_ffi.LINEAR_PLAN_PLAIN) == BAD  # the plan's alone


def test_every_count_that_a_field_would_cut_off_is_refused():
    """Plans and workspace sizes too, and 64-bit counts: a workspace of -1 bytes
    would pass for one of 2**64 - 1."""
    for bad in (1 << 32, (1 << 32) + 1, -1):
        for call in (lambda: hx.linear_plan("forward", bad, 64, 64),
                     lambda: hx.linear_plan("weight_grad", 64, 64, bad),
                     lambda: hx.linear_plan("forward", 64, 64, 64, flags=bad),
                     lambda: hx.grad_workspace_bytes(bad)):
            with pytest.raises(ValueError):
                call()
    for bad in (1 << 64, (1 << 64) + 3, -1):
        for call in (lambda: hx.cuda_layer_norm(0, P, P, bad, 8),
                     lambda: hx.cuda_layer_norm_grad(0, P, P, P, P, P, bad, 8),
                     lambda: hx.cuda_layer_norm_grad(0, P, P, P, P, P, 8, 8, dbeta=P,
                                                     workspace=P, workspace_bytes=bad),
                     lambda: hx.cuda_linear_output_grad(0, P, 8, 8, dbias=P, workspace=P,
                                                        workspace_bytes=bad)):
            with pytest.raises(ValueError):
                call()
