"""The layer calls (include/hexir_b200/layers.h) on a B200 against their
definitions in 64 bits (tests/layers_reference.py holds the formulas and the
derived bounds; every element is compared).

Outputs lie inside buffers filled with a pattern, with rows padded where a
stride is wider than the row; everything around an output must keep it.
"""

import numpy as np
import pytest
import torch

import hexir_b200 as hx
from hexir_b200 import _ffi
from tests import layers_reference as ref

pytestmark = pytest.mark.gpu

TORCH = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16,
         "f16": torch.float16}
FILL = 77.0
GUARD = 512


class Tensor:
    """rows x cols at a row stride of cols + pad, `shift` elements into a
    buffer, with GUARD elements before and after."""

    def __init__(self, rows, cols, dtype, pad=0, shift=0, data=None):
        self.rows, self.cols, self.ld = rows, cols, cols + pad
        self.start = GUARD + shift
        span = max(rows - 1, 0) * self.ld + (cols if rows else 0)
        self.flat = torch.full((self.start + span + GUARD,), FILL, device="cuda",
                               dtype=TORCH[dtype])
        self.view = self.flat.as_strided((rows, cols), (self.ld, 1), self.start)
        if data is not None:
            self.view.copy_(torch.as_tensor(data).reshape(rows, cols))

    @property
    def ptr(self):
        return self.view.data_ptr() if self.view.numel() else self.flat.data_ptr()

    def numpy(self):
        return self.view.double().cpu().numpy()

    def check_frame(self):
        rest = self.flat.clone()
        rest.as_strided((self.rows, self.cols), (self.ld, 1), self.start).fill_(FILL)
        assert bool((rest == FILL).all()), "a write outside the output"


def normal(rng, shape, scale=1.0):
    return rng.standard_normal(shape) * scale


def inputs(rng, rows, cols, dtype, pad=0, shift=0, scale=1.0, mean=0.0):
    return Tensor(rows, cols, dtype, pad, shift,
                  normal(rng, (rows, cols), scale) + mean)


def sync():
    hx.cuda_synchronize(0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


def stream():
    return torch.cuda.current_stream().cuda_stream


def assert_within(got, want, bound, what):
    off = np.abs(got - want) - bound
    bad = ~(off <= 0)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(
            f"{what}: {bad.sum()} of {bad.size} out of bound, first at {at}: got "
            f"{got[at]!r}, want {want[at]!r} +- {bound[at]!r}")


# ----------------------------------------------------------------- layer norm

NORM_SHAPES = [  # every kernel's row length, at and around its limits
    (1, 1), (3, 2), (5, 7), (9, 64), (33, 255), (17, 256), (8, 257), (6, 512),
    (19, 1000), (11, 1024), (7, 1025), (301, 2048), (5, 2049), (4, 4096),
    (3, 4104), (3, 8192), (2, 8193), (2, 16384), (2, 16385), (3, 20000)]


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 8), (3, 1)])
def test_layer_norm(rows, cols, dtype, pad, shift):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = inputs(rng, rows, cols, dtype, pad, shift, 2.0, 3.0)
    gamma = inputs(rng, 1, cols, dtype, shift=shift, scale=0.2, mean=1.0)
    beta = inputs(rng, 1, cols, dtype, shift=shift, scale=0.2)
    wide = "f64" if dtype == "f64" else "f32"
    y = Tensor(rows, cols, dtype, pad, shift)
    mean, rstd = Tensor(1, rows, wide), Tensor(1, rows, wide)
    hx.cuda_layer_norm(0, x.ptr, y.ptr, rows, cols, dtype, gamma=gamma.ptr,
                       beta=beta.ptr, mean=mean.ptr, rstd=rstd.ptr, eps=1e-5,
                       ldx=x.ld, ldy=y.ld, stream=stream())
    sync()
    want = ref.layer_norm(x.numpy(), gamma.numpy()[0], beta.numpy()[0], 1e-5, dtype)
    for t in (y, mean, rstd):
        t.check_frame()
    for got, (w, bound), what in ((y.numpy(), want[0], "y"),
                                  (mean.numpy()[0], want[1], "mean"),
                                  (rstd.numpy()[0], want[2], "rstd")):
        assert_within(got, w, bound, what)


@pytest.mark.parametrize("dtype", ["f64", "bf16"])
@pytest.mark.parametrize("cols", [40, 1024, 3000, 17000])
def test_layer_norm_without_parameters_in_place(dtype, cols):
    rng = np.random.default_rng(cols)
    x = inputs(rng, 5, cols, dtype, mean=-1.0)
    before = x.numpy()
    hx.cuda_layer_norm(0, x.ptr, x.ptr, 5, cols, dtype, eps=0.25, stream=stream())
    sync()
    x.check_frame()
    (want, bound), _, _ = ref.layer_norm(before, None, None, 0.25, dtype)
    assert_within(x.numpy(), want, bound, "y")


@pytest.mark.parametrize("cols", [8, 1000, 5000, 20000])
def test_layer_norm_of_constant_and_special_rows(cols):
    """A constant row has variance 0 (y = beta); a NaN or an infinity makes its
    own row NaN and no other."""
    x = torch.randn(6, cols, device="cuda")
    x[1] = 3.0
    x[2, cols // 2] = float("nan")
    x[4, 0] = float("inf")
    y = torch.empty_like(x)
    beta = torch.randn(cols, device="cuda")
    hx.cuda_layer_norm(0, x.data_ptr(), y.data_ptr(), 6, cols, "f32",
                       beta=beta.data_ptr(), eps=1e-5, stream=stream())
    sync()
    assert bool((y[1] == beta).all())
    assert bool(y[2].isnan().all()) and bool(y[4].isnan().all())
    assert bool(y[[0, 1, 3, 5]].isfinite().all())


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(1000, 96), (2000, 768)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 8), (3, 1)])
def test_layer_norm_grad(rows, cols, dtype, pad, shift):
    rng = np.random.default_rng(rows + 7 * cols)
    wide = "f64" if dtype == "f64" else "f32"
    dy = inputs(rng, rows, cols, dtype, pad, shift)
    x = inputs(rng, rows, cols, dtype, pad, shift, 2.0, 1.0)
    residual = inputs(rng, rows, cols, dtype, pad, shift)
    gamma = inputs(rng, 1, cols, dtype, shift=shift, scale=0.2, mean=1.0)
    xd = x.numpy()
    mean = Tensor(1, rows, wide, data=xd.mean(1))
    rstd = Tensor(1, rows, wide, data=1 / np.sqrt(xd.var(1) + 1e-3))
    dx = Tensor(rows, cols, dtype, pad, shift)
    dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
    size = hx.grad_workspace_bytes(cols, dtype)
    work = torch.full((size + 64,), 0xA5, device="cuda", dtype=torch.uint8)
    hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, dx.ptr, rows, cols,
                            dtype, gamma=gamma.ptr, dgamma=dgamma.ptr,
                            dbeta=dbeta.ptr, residual=residual.ptr,
                            workspace=work.data_ptr(), workspace_bytes=size,
                            lddy=dy.ld, ldx=x.ld, lddx=dx.ld, ldr=residual.ld,
                            stream=stream())
    sync()
    want = ref.layer_norm_grad(dy.numpy(), xd, mean.numpy()[0], rstd.numpy()[0],
                               gamma.numpy()[0], residual.numpy(), dtype)
    for t in (dx, dgamma, dbeta):
        t.check_frame()
    assert bool((work[size:] == 0xA5).all()), "a write behind the workspace"
    for got, (w, bound), what in ((dx.numpy(), want[0], "dx"),
                                  (dgamma.numpy()[0], want[1], "dgamma"),
                                  (dbeta.numpy()[0], want[2], "dbeta")):
        assert_within(got, w, bound, what)


# ------------------------------------------------------------------- products

GUARDED, SINGLE, PAIR, SKINNY = (_ffi.LINEAR_FORCE_GUARDED, _ffi.LINEAR_FORCE_SINGLE,
                                 _ffi.LINEAR_FORCE_PAIR, _ffi.LINEAR_FORCE_SKINNY)
# (m, n, k): one tile, partial tiles on each side, several tiles, an odd
# number of pairs, sums of one and of many stages, single rows and columns.
SHAPES = [(128, 128, 64), (1, 1, 1), (1, 8, 8), (8, 1, 8), (129, 136, 72),
          (100, 264, 200), (256, 256, 640), (300, 520, 1000), (513, 72, 2056),
          (777, 1001, 153), (64, 300, 512)]


def linear_case(m, n, k, dtype, act, flags, pad=0, shift=0, bias=True, residual=True,
                preact=True, seed=0):
    rng = np.random.default_rng(m * 7 + n * 3 + k + seed)
    x = inputs(rng, m, k, dtype, pad, shift)
    w = inputs(rng, k, n, dtype, pad, shift, scale=1 / np.sqrt(max(k, 1)))
    b = inputs(rng, 1, n, dtype, shift=shift) if bias else None
    r = inputs(rng, m, n, dtype, pad, shift) if residual else None
    y = Tensor(m, n, dtype, pad, shift)
    z = Tensor(m, n, dtype, pad, shift) if preact else None
    hx.cuda_linear(0, x.ptr, w.ptr, y.ptr, m, n, k, dtype, act,
                   bias=b.ptr if b else 0, residual=r.ptr if r else 0,
                   preact=z.ptr if z else 0, ldx=x.ld, ldw=w.ld, ldy=y.ld,
                   ldr=r.ld if r else 0, ldp=z.ld if z else 0, flags=flags,
                   stream=stream())
    sync()
    want = ref.linear(x.numpy(), w.numpy(), b.numpy()[0] if b else None, act,
                      r.numpy() if r else None, dtype)
    y.check_frame()
    assert_within(y.numpy(), want[0], want[1], "y")
    if z:
        z.check_frame()
        assert_within(z.numpy(), want[2], want[3], "z")
    return y, z


def aligned8(*sizes):
    return all(s % 8 == 0 for s in sizes)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("split", [1, 2, 8])
@pytest.mark.parametrize("dtype,pad,shift", [("bf16", 0, 0), ("f16", 5, 3),
                                             ("bf16", 2, 2)])
def test_linear_guarded(m, n, k, dtype, split, pad, shift):
    linear_case(m, n, k, dtype, "gelu", GUARDED | _ffi.LINEAR_SPLIT(split), pad, shift)


@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if aligned8(s[1], s[2])])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 24)])
def test_linear_single(m, n, k, dtype, split, pad):
    linear_case(m, n, k, dtype, "swish", SINGLE | _ffi.LINEAR_SPLIT(split), pad)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("n,k", [(8, 8), (136, 72), (1000, 1032), (512, 4096)])
@pytest.mark.parametrize("split", [1, 2, 8])
@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 8)])
def test_linear_skinny(m, n, k, dtype, split, pad):
    linear_case(m, n, k, dtype, "tanh", SKINNY | _ffi.LINEAR_SPLIT(split), pad)


@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if aligned8(s[1], s[2])]
                         + [(1100, 2600, 192), (2600, 4000, 64)])
@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 24)])
def test_linear_pair(m, n, k, dtype, pad):
    linear_case(m, n, k, dtype, "none", PAIR, pad)


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(5, 200, 64), (200, 336, 128), (70, 99, 65)])
def test_linear_chosen_kernel_and_activations(m, n, k, dtype, act):
    linear_case(m, n, k, dtype, act, 0)
    linear_case(m, n, k, dtype, act, 0, bias=False, residual=False, preact=False)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("flags", [0, GUARDED | _ffi.LINEAR_SPLIT(2), SINGLE,
                                   SINGLE | _ffi.LINEAR_SPLIT(4), PAIR])
@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 8)])
def test_linear_input_grad(m, n, k, dtype, pad, flags):
    if flags & (SINGLE | PAIR) and not aligned8(n + pad):
        pytest.skip("TMA kernels need aligned rows")
    rng = np.random.default_rng(m + n + k)
    dz = inputs(rng, m, n, dtype, pad)
    w = inputs(rng, k, n, dtype, pad, scale=1 / np.sqrt(n))
    prev, r = inputs(rng, m, k, dtype, pad), inputs(rng, m, k, dtype, pad)
    for act, residual in (("gelu", r), ("none", None), ("mish", r)):
        dx = Tensor(m, k, dtype, pad)
        hx.cuda_linear_input_grad(0, dz.ptr, w.ptr, dx.ptr, m, n, k, dtype, act,
                                  preact=prev.ptr, residual=residual.ptr if residual else 0,
                                  lddz=dz.ld, ldw=w.ld, lddx=dx.ld, ldp=prev.ld,
                                  ldr=r.ld, flags=flags, stream=stream())
        sync()
        dx.check_frame()
        want = ref.product(dz.numpy(), w.numpy().T, dtype, act, prev.numpy(),
                           residual.numpy() if residual else None)
        assert_within(dx.numpy(), *want, "dx")


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("flags", [0, GUARDED | _ffi.LINEAR_SPLIT(2), SINGLE,
                                   SINGLE | _ffi.LINEAR_SPLIT(4), PAIR])
@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 8)])
def test_linear_weight_grad(m, n, k, dtype, pad, flags):
    if flags & (SINGLE | PAIR) and not aligned8(n + pad, k + pad):
        pytest.skip("TMA kernels need aligned rows")
    rng = np.random.default_rng(m + 2 * n + k)
    x, dz = inputs(rng, m, k, dtype, pad), inputs(rng, m, n, dtype, pad)
    dw = Tensor(k, n, dtype, pad)
    hx.cuda_linear_weight_grad(0, x.ptr, dz.ptr, dw.ptr, m, n, k, dtype, ldx=x.ld,
                               lddz=dz.ld, lddw=dw.ld, flags=flags, stream=stream())
    sync()
    dw.check_frame()
    assert_within(dw.numpy(), *ref.product(x.numpy().T, dz.numpy(), dtype), "dw")


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("dtype,pad,shift", [("bf16", 0, 0), ("f16", 8, 8),
                                             ("bf16", 3, 1)])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 8), (70, 250), (33, 256), (1000, 264),
                                 (5000, 24)])
def test_linear_output_grad(m, n, dtype, act, pad, shift):
    rng = np.random.default_rng(m * n)
    dy, z = inputs(rng, m, n, dtype, pad, shift), inputs(rng, m, n, dtype, pad, shift, 3.0)
    dz, dbias = Tensor(m, n, dtype, pad, shift), Tensor(1, n, dtype)
    size = hx.grad_workspace_bytes(n, dtype)
    work = torch.full((size + 64,), 0xA5, device="cuda", dtype=torch.uint8)
    hx.cuda_linear_output_grad(0, dy.ptr, m, n, dtype, act, preact=z.ptr, dz=dz.ptr,
                               dbias=dbias.ptr, workspace=work.data_ptr(),
                               workspace_bytes=size, lddy=dy.ld, ldp=z.ld, lddz=dz.ld,
                               stream=stream())
    sync()
    dz.check_frame()
    dbias.check_frame()
    assert bool((work[size:] == 0xA5).all()), "a write behind the workspace"
    assert_within(dz.numpy(), *ref.output_grad(dy.numpy(), z.numpy(), act, dtype), "dz")
    assert_within(dbias.numpy()[0], *ref.column_sums(dz.numpy(), dtype), "dbias")
