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


# ------------------------------------------------- forms, streams and captures

def forced(m, n, k):
    """Every kernel that can run the shape, by flags."""
    out = [0, GUARDED | _ffi.LINEAR_SPLIT(1), GUARDED | _ffi.LINEAR_SPLIT(2)]
    if aligned8(n, k):
        out += [SINGLE | _ffi.LINEAR_TILE(64) | _ffi.LINEAR_SPLIT(1),
                SINGLE | _ffi.LINEAR_TILE(64) | _ffi.LINEAR_SPLIT(4),
                PAIR | _ffi.LINEAR_TILE(128), PAIR | _ffi.LINEAR_TILE(256)]
        if m <= 64:
            out += [SKINNY | _ffi.LINEAR_SPLIT(1), SKINNY | _ffi.LINEAR_SPLIT(4)]
    return out


@pytest.mark.parametrize("m,n,k", [(48, 200, 304), (300, 520, 136), (70, 99, 65)])
def test_every_kernel_in_place_over_the_residual(m, n, k):
    """y may be the residual's own buffer; every tile width too."""
    rng = np.random.default_rng(k)
    x = inputs(rng, m, k, "bf16")
    w = inputs(rng, k, n, "bf16", scale=1 / np.sqrt(k))
    start = normal(rng, (m, n))
    for flags in forced(m, n, k):
        y = Tensor(m, n, "bf16", data=start)
        r = y.numpy()
        hx.cuda_linear(0, x.ptr, w.ptr, y.ptr, m, n, k, "bf16", "gelu",
                       residual=y.ptr, flags=flags, stream=stream())
        sync()
        y.check_frame()
        want = ref.linear(x.numpy(), w.numpy(), None, "gelu", r, "bf16")
        assert_within(y.numpy(), want[0], want[1], f"flags {flags:#x}")


@pytest.mark.parametrize("ldx,ldw,ldy", [(136, 257, 256), (135, 256, 256),
                                         (136, 256, 257), (129, 250, 249)])
def test_operands_by_tma_and_by_guarded_loads_mix(ldx, ldw, ldy):
    """One operand on 16-byte rows, the other (or the output) off them."""
    m, n, k = 200, 249, 129
    rng = np.random.default_rng(ldx + ldw)
    x = Tensor(m, k, "f16", ldx - k, data=normal(rng, (m, k)))
    w = Tensor(k, n, "f16", ldw - n, data=normal(rng, (k, n), 1 / np.sqrt(k)))
    r = Tensor(m, n, "f16", ldy - n, data=normal(rng, (m, n)))
    y = Tensor(m, n, "f16", ldy - n)
    hx.cuda_linear(0, x.ptr, w.ptr, y.ptr, m, n, k, "f16", "swish", residual=r.ptr,
                   ldx=ldx, ldw=ldw, ldy=ldy, ldr=ldy, stream=stream())
    sync()
    y.check_frame()
    want = ref.linear(x.numpy(), w.numpy(), None, "swish", r.numpy(), "f16")
    assert_within(y.numpy(), want[0], want[1], "y")


def test_empty_sums_and_empty_outputs():
    b, r = inputs(np.random.default_rng(1), 1, 40, "bf16"), \
        inputs(np.random.default_rng(2), 7, 40, "bf16")
    y, z = Tensor(7, 40, "bf16"), Tensor(7, 40, "bf16")
    hx.cuda_linear(0, 0, 0, y.ptr, 7, 40, 0, "bf16", "tanh", bias=b.ptr,
                   residual=r.ptr, preact=z.ptr, stream=stream())
    sync()
    want = ref.linear(np.zeros((7, 0)), np.zeros((0, 40)), b.numpy()[0], "tanh",
                      r.numpy(), "bf16")
    assert_within(y.numpy(), want[0], want[1], "y")
    assert_within(z.numpy(), want[2], want[3], "z")
    y.check_frame()
    # No output, or none of it: nothing is written, nothing is needed.
    for m, n in ((0, 40), (7, 0), (0, 0)):
        hx.cuda_linear(0, 0, 0, 0, m, n, 16, stream=stream())
        hx.cuda_linear_output_grad(0, 0, m, n, "bf16", "gelu", stream=stream())
    hx.cuda_linear_input_grad(0, 0, 0, 0, 0, 8, 8, stream=stream())
    # Sums over no rows are zeros.
    dw, db = Tensor(24, 40, "f16"), Tensor(1, 40, "f16")
    work = torch.empty(hx.grad_workspace_bytes(40, "f16"), device="cuda",
                       dtype=torch.uint8)
    hx.cuda_linear_weight_grad(0, 0, 0, dw.ptr, 0, 40, 24, "f16", stream=stream())
    hx.cuda_linear_output_grad(0, 0, 0, 40, "f16", dbias=db.ptr,
                               workspace=work.data_ptr(),
                               workspace_bytes=work.numel(), stream=stream())
    # dz . w^T over no columns of dz is the residual.
    dx, res = Tensor(5, 24, "f16"), inputs(np.random.default_rng(3), 5, 24, "f16")
    hx.cuda_linear_input_grad(0, 0, 0, dx.ptr, 5, 0, 24, "f16", residual=res.ptr,
                              stream=stream())
    dg, dbeta = Tensor(1, 40, "f64"), Tensor(1, 40, "f64")
    work64 = torch.empty(hx.grad_workspace_bytes(40, "f64"), device="cuda",
                         dtype=torch.uint8)
    hx.cuda_layer_norm(0, 0, 0, 0, 40, "f32", stream=stream())
    hx.cuda_layer_norm_grad(0, 0, 0, 0, 0, 0, 0, 40, "f64", dgamma=dg.ptr,
                            dbeta=dbeta.ptr, workspace=work64.data_ptr(),
                            workspace_bytes=work64.numel(), stream=stream())
    sync()
    for t in (dw, db, dg, dbeta):
        t.check_frame()
        assert not t.numpy().any()
    assert np.array_equal(dx.numpy(), res.numpy())


@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("bf16", 1001), ("f32", 4096),
                                        ("f64", 1025), ("f16", 20000)])
def test_layer_norm_grad_in_place(dtype, cols):
    """dx may be dy, or the residual; sums alone and dx alone."""
    rng = np.random.default_rng(cols)
    rows, wide = 37, "f64" if dtype == "f64" else "f32"
    x = inputs(rng, rows, cols, dtype)
    mean = Tensor(1, rows, wide, data=x.numpy().mean(1))
    rstd = Tensor(1, rows, wide, data=1 / np.sqrt(x.numpy().var(1) + 1e-3))
    dy0, r0 = normal(rng, (rows, cols)), normal(rng, (rows, cols))
    size = hx.grad_workspace_bytes(cols, dtype)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)
    for place in ("dy", "residual", "sums"):
        dy, r = Tensor(rows, cols, dtype, data=dy0), Tensor(rows, cols, dtype, data=r0)
        want = ref.layer_norm_grad(dy.numpy(), x.numpy(), mean.numpy()[0],
                                   rstd.numpy()[0], None, r.numpy(), dtype)
        dx = {"dy": dy, "residual": r, "sums": None}[place]
        dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
        hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr,
                                dx.ptr if dx else 0, rows, cols, dtype,
                                dgamma=dgamma.ptr, dbeta=dbeta.ptr, residual=r.ptr,
                                workspace=work.data_ptr(), workspace_bytes=size,
                                stream=stream())
        sync()
        assert_within(dgamma.numpy()[0], *want[1], "dgamma")
        assert_within(dbeta.numpy()[0], *want[2], "dbeta")
        if dx:
            assert_within(dx.numpy(), *want[0], "dx")
        else:
            dx = Tensor(rows, cols, dtype)
            hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, dx.ptr, rows,
                                    cols, dtype, residual=r.ptr, stream=stream())
            sync()
            assert_within(dx.numpy(), *want[0], "dx")


def test_output_grad_in_place_and_alone():
    rng = np.random.default_rng(9)
    z, dy = inputs(rng, 90, 72, "bf16"), inputs(rng, 90, 72, "bf16")
    want = ref.output_grad(dy.numpy(), z.numpy(), "swish", "bf16")
    hx.cuda_linear_output_grad(0, dy.ptr, 90, 72, "bf16", "swish", preact=z.ptr,
                               dz=dy.ptr, stream=stream())
    sync()
    dy.check_frame()
    assert_within(dy.numpy(), *want, "dz")


@pytest.mark.parametrize("flags", [0, GUARDED, PAIR, SKINNY])
def test_a_nan_stays_in_its_row_and_column(flags):
    m, n, k = 40, 264, 200
    rng = np.random.default_rng(4)
    x = torch.tensor(normal(rng, (m, k)), device="cuda").bfloat16()
    w = torch.tensor(normal(rng, (k, n)), device="cuda").bfloat16()
    x[3, 7], x[20, k - 1] = float("nan"), float("inf")
    w[k - 1, 100] = float("nan")
    y = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    hx.cuda_linear(0, x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k,
                   flags=flags, stream=stream())
    sync()
    fine = torch.ones(m, n, dtype=torch.bool, device="cuda")
    fine[3], fine[20], fine[:, 100] = False, False, False
    assert bool(y[fine].isfinite().all())
    assert bool(y[3].isnan().all()) and bool(y[:, 100].isnan().all())
    assert not bool(y[20].isfinite().any())


def test_offsets_beyond_32_bits():
    """Row strides that put the last rows past 2^32 elements."""
    rows, cols, ld = 4, 1000, 1_500_000_064
    big = torch.empty(3 * ld + cols, device="cuda", dtype=torch.bfloat16)
    x = big.as_strided((rows, cols), (ld, 1))
    x.copy_(torch.randn(rows, cols, device="cuda"))
    y = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    hx.cuda_layer_norm(0, x.data_ptr(), y.data_ptr(), rows, cols, "bf16", ldx=ld,
                       stream=stream())
    sync()
    (want, bound), _, _ = ref.layer_norm(x.double().cpu().numpy(), None, None, 1e-5,
                                         "bf16")
    assert_within(y.double().cpu().numpy(), want, bound, "y")
    w = torch.randn(cols, 64, device="cuda").bfloat16()
    out = torch.empty(rows, 64, device="cuda", dtype=torch.bfloat16)
    res = x[:, :64]
    for flags in (0, GUARDED, SINGLE, PAIR):
        hx.cuda_linear(0, x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, 64, cols,
                       "bf16", residual=res.data_ptr(), ldx=ld, ldr=ld, flags=flags,
                       stream=stream())
        sync()
        want = ref.linear(x.double().cpu().numpy(), w.double().cpu().numpy(), None,
                          "none", res.double().cpu().numpy(), "bf16")
        assert_within(out.double().cpu().numpy(), want[0], want[1], f"y {flags:#x}")


def feed_forward(rows, cols, hidden, dtype="bf16", seed=0):
    """A pre-norm feed-forward block's tensors, as torch tensors."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TORCH[dtype]

    def normal_(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)
    return {"x": normal_(rows, cols), "gamma": normal_(cols, std=0.1, mean=1.0),
            "beta": normal_(cols, std=0.1),
            "w1": normal_(cols, hidden, std=cols ** -0.5), "b1": normal_(hidden, std=0.1),
            "w2": normal_(hidden, cols, std=hidden ** -0.5), "b2": normal_(cols, std=0.1),
            "dy": normal_(rows, cols)}


class Block:
    """y = x + w2 . gelu(w1 . norm(x) + b1) + b2 and all its gradients through the
    layer calls, in buffers made once."""

    def __init__(self, rows, cols, hidden, dtype="bf16"):
        self.shape, self.dtype = (rows, cols, hidden), dtype
        t = TORCH[dtype]

        def empty(*shape, of=t):
            return torch.empty(*shape, device="cuda", dtype=of)
        self.h, self.dh, self.dx = (empty(rows, cols) for _ in range(3))
        self.a, self.z, self.dz = (empty(rows, hidden) for _ in range(3))
        self.y = empty(rows, cols)
        self.mean, self.rstd = (empty(rows, of=torch.float32) for _ in range(2))
        self.dw1, self.dw2 = empty(cols, hidden), empty(hidden, cols)
        self.db1, self.db2 = empty(hidden), empty(cols)
        self.dgamma, self.dbeta = empty(cols), empty(cols)
        self.work = empty(hx.grad_workspace_bytes(max(cols, hidden), dtype),
                          of=torch.uint8)

    def forward(self, p, on):
        r, c, f = self.shape
        hx.cuda_layer_norm(0, p["x"].data_ptr(), self.h.data_ptr(), r, c, self.dtype,
                           gamma=p["gamma"].data_ptr(), beta=p["beta"].data_ptr(),
                           mean=self.mean.data_ptr(), rstd=self.rstd.data_ptr(),
                           stream=on)
        hx.cuda_linear(0, self.h.data_ptr(), p["w1"].data_ptr(), self.a.data_ptr(), r, f,
                       c, self.dtype, "gelu", bias=p["b1"].data_ptr(),
                       preact=self.z.data_ptr(), stream=on)
        hx.cuda_linear(0, self.a.data_ptr(), p["w2"].data_ptr(), self.y.data_ptr(), r, c,
                       f, self.dtype, bias=p["b2"].data_ptr(),
                       residual=p["x"].data_ptr(), stream=on)

    def backward(self, p, on):
        r, c, f = self.shape
        dt, work = self.dtype, self.work
        dy = p["dy"].data_ptr()
        hx.cuda_linear_output_grad(0, dy, r, c, dt, dbias=self.db2.data_ptr(),
                                   workspace=work.data_ptr(),
                                   workspace_bytes=work.numel(), stream=on)
        hx.cuda_linear_weight_grad(0, self.a.data_ptr(), dy, self.dw2.data_ptr(), r, c,
                                   f, dt, stream=on)
        hx.cuda_linear_input_grad(0, dy, p["w2"].data_ptr(), self.dz.data_ptr(), r, c, f,
                                  dt, "gelu", preact=self.z.data_ptr(), stream=on)
        hx.cuda_linear_output_grad(0, self.dz.data_ptr(), r, f, dt,
                                   dbias=self.db1.data_ptr(), workspace=work.data_ptr(),
                                   workspace_bytes=work.numel(), stream=on)
        hx.cuda_linear_weight_grad(0, self.h.data_ptr(), self.dz.data_ptr(),
                                   self.dw1.data_ptr(), r, f, c, dt, stream=on)
        hx.cuda_linear_input_grad(0, self.dz.data_ptr(), p["w1"].data_ptr(),
                                  self.dh.data_ptr(), r, f, c, dt, stream=on)
        hx.cuda_layer_norm_grad(0, self.dh.data_ptr(), p["x"].data_ptr(),
                                self.mean.data_ptr(), self.rstd.data_ptr(),
                                self.dx.data_ptr(), r, c, dt,
                                gamma=p["gamma"].data_ptr(),
                                dgamma=self.dgamma.data_ptr(),
                                dbeta=self.dbeta.data_ptr(), residual=dy,
                                workspace=work.data_ptr(),
                                workspace_bytes=work.numel(), stream=on)

    def outputs(self):
        return {"y": self.y, "dx": self.dx, "dw1": self.dw1, "dw2": self.dw2,
                "db1": self.db1, "db2": self.db2, "dgamma": self.dgamma,
                "dbeta": self.dbeta}


def block_in_64_bits(p):
    q = {k: v.double().requires_grad_(k != "dy") for k, v in p.items()}
    x = q["x"]
    mean = x.mean(1, keepdim=True)
    h = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    z = (h * q["gamma"] + q["beta"]) @ q["w1"] + q["b1"]
    a = 0.5 * z * torch.erfc(-z * 0.5 ** 0.5)
    y = x + a @ q["w2"] + q["b2"]
    y.backward(q["dy"])
    names = {"dx": "x", "dw1": "w1", "dw2": "w2", "db1": "b1", "db2": "b2",
             "dgamma": "gamma", "dbeta": "beta"}
    return {"y": y.detach(), **{k: q[v].grad for k, v in names.items()}}


def worst(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("rows,cols,hidden", [(300, 256, 1024), (1, 512, 2048),
                                              (77, 130, 515)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_feed_forward_block_forward_and_backward(rows, cols, hidden, dtype):
    """The calls in a row, as a training step has them.  Every stage stores its
    result in the type, off by a half step at most: the relative error of an
    output is that of the 7 roundings before it, each carried on by products
    whose norms the next stage's stay within, so 7 half steps and one for
    their second order bound it in the 2-norm (the roundings are far from
    aligned; the products' f32 sums are 2^-15 below them)."""
    p = feed_forward(rows, cols, hidden, dtype)
    block = Block(rows, cols, hidden, dtype)
    block.forward(p, stream())
    block.backward(p, stream())
    sync()
    want = block_in_64_bits(p)
    for name, got in block.outputs().items():
        assert worst(got, want[name]) <= 8 * ref.HALF[dtype], name


def test_a_captured_training_step_replays():
    """A block's step captured into a graph: replays follow its inputs, equal
    the same calls made eagerly bit for bit, and two graphs with workspaces of
    their own run side by side on two streams."""
    shape = (260, 256, 1000)
    eager = Block(*shape)
    p = feed_forward(*shape, seed=1)
    eager.forward(p, stream())       # also: the device code is loaded
    eager.backward(p, stream())
    sync()
    steps = []
    for seed in (1, 2):
        mine, block, on = feed_forward(*shape, seed=seed), Block(*shape), torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=on):
            s = torch.cuda.current_stream().cuda_stream
            block.forward(mine, s)
            block.backward(mine, s)
        steps.append((mine, block, on, graph))
    for seeds in ((1, 2), (5, 6), (7, 8)):
        for (mine, block, on, graph), seed in zip(steps, seeds):
            fresh = feed_forward(*shape, seed=seed)
            torch.cuda.synchronize()
            for k in mine:
                mine[k].copy_(fresh[k])
        torch.cuda.synchronize()
        for mine, block, on, graph in steps:
            with torch.cuda.stream(on):
                graph.replay()
                graph.replay()
        sync()
        for mine, block, on, graph in steps:
            eager.forward(mine, stream())
            eager.backward(mine, stream())
            sync()
            for (name, got), want in zip(block.outputs().items(),
                                         eager.outputs().values()):
                assert torch.equal(got, want), name


def test_streams_and_threads_at_once():
    """The same step from four threads, each on a stream of its own: every
    result has the bits of the step made alone."""
    import threading
    shape = (200, 256, 600)
    inputs_ = [feed_forward(*shape, seed=s) for s in range(4)]
    alone = []
    for p in inputs_:
        b = Block(*shape)
        b.forward(p, stream())
        b.backward(p, stream())
        sync()
        alone.append(b)
    blocks, streams = [Block(*shape) for _ in range(4)], [torch.cuda.Stream()
                                                         for _ in range(4)]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            for _ in range(10):
                blocks[i].forward(inputs_[i], streams[i].cuda_stream)
                blocks[i].backward(inputs_[i], streams[i].cuda_stream)
        except Exception as err:  # noqa: BLE001 - reported below
            errors.append(err)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    sync()
    assert not errors
    for a, b in zip(alone, blocks):
        for (name, got), want in zip(b.outputs().items(), a.outputs().values()):
            assert torch.equal(got, want), name


def test_results_repeat_bit_for_bit():
    """Sums have a fixed order: the same call twice, in between other work."""
    p = feed_forward(513, 768, 1030, seed=3)
    first, second = Block(513, 768, 1030), Block(513, 768, 1030)
    for b in (first, second):
        b.forward(p, stream())
        b.backward(p, stream())
        Block(5, 64, 64).forward(feed_forward(5, 64, 64), stream())
    sync()
    for (name, a), b in zip(first.outputs().items(), second.outputs().values()):
        assert torch.equal(a, b), name


def test_gradients_against_differences():
    """The block's gradient along a direction, against a difference of its loss
    sum(y dy) in 64 bits: the gradient is in f16 (2^-11 a rounding, 8 of them),
    the difference is off by its step's square (1e-8 of the third derivative)."""
    p = feed_forward(20, 64, 128, "f16", seed=4)
    block = Block(20, 64, 128, "f16")
    block.forward(p, stream())
    block.backward(p, stream())
    sync()

    def loss(q):
        x = q["x"]
        mean = x.mean(1, keepdim=True)
        h = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
        z = (h * q["gamma"] + q["beta"]) @ q["w1"] + q["b1"]
        return ((x + 0.5 * z * torch.erfc(-z * 0.5 ** 0.5) @ q["w2"] + q["b2"])
                * q["dy"]).sum()
    names = {"x": "dx", "w1": "dw1", "w2": "dw2", "b1": "db1", "b2": "db2",
             "gamma": "dgamma", "beta": "dbeta"}
    q = {k: v.double() for k, v in p.items()}
    for name, grad in names.items():
        g = getattr(block, grad).double()
        along = g / g.norm()  # the gradient's own direction: no cancellation
        step = 1e-4
        up, down = dict(q), dict(q)
        up[name], down[name] = q[name] + step * along, q[name] - step * along
        slope = float((loss(up) - loss(down)) / (2 * step))
        assert abs(slope - float(g.norm())) <= (8 * ref.HALF["f16"] + 1e-6) * abs(slope)


def test_launch_faults_are_reported_and_leave_nothing_behind():
    x = torch.randn(64, 64, device="cuda").bfloat16()
    y = torch.empty_like(x)
    before = hx.launch_count()
    hx.fault_configure("launch:1")
    try:
        with pytest.raises(_ffi.HexirError) as err:
            hx.cuda_linear(0, x.data_ptr(), x.data_ptr(), y.data_ptr(), 64, 64, 64,
                           stream=stream())
        assert err.value.status == _ffi.ERROR_DEVICE
    finally:
        hx.fault_configure("")
    hx.cuda_linear(0, x.data_ptr(), x.data_ptr(), y.data_ptr(), 64, 64, 64,
                   stream=stream())
    sync()
    assert hx.launch_count() == before + 1
    with pytest.raises(_ffi.HexirError) as err:
        hx.cuda_layer_norm(99, x.data_ptr(), y.data_ptr(), 64, 64, "bf16")
    assert err.value.status == _ffi.ERROR_DEVICE


@pytest.mark.parametrize("rows,cols", [(2200, 2296), (2560, 1928), (1000, 5136)])
def test_pairs_that_cut_the_last_tiles_in_two(rows, cols):
    """More 256 x 256 tiles than CTA pairs by a few: the last ones are halves,
    one of them possibly beyond the columns."""
    depth, flags = 136, PAIR | _ffi.LINEAR_TILE(256)
    rng = np.random.default_rng(cols)
    a, b = inputs(rng, rows, depth, "bf16"), inputs(rng, depth, cols, "bf16", scale=0.1)
    bt, at = Tensor(cols, depth, "bf16", data=b.numpy().T), \
        Tensor(depth, rows, "bf16", data=a.numpy().T)
    r, z = inputs(rng, rows, cols, "bf16"), Tensor(rows, cols, "bf16")
    bias = inputs(rng, 1, cols, "bf16")
    y, dx, dw = (Tensor(rows, cols, "bf16") for _ in range(3))
    on = stream()
    hx.cuda_linear(0, a.ptr, b.ptr, y.ptr, rows, cols, depth, "bf16", "tanh",
                   bias=bias.ptr, residual=r.ptr, preact=z.ptr, flags=flags, stream=on)
    hx.cuda_linear_input_grad(0, a.ptr, bt.ptr, dx.ptr, rows, depth, cols, "bf16",
                              "swish", preact=r.ptr, flags=flags, stream=on)
    hx.cuda_linear_weight_grad(0, at.ptr, b.ptr, dw.ptr, depth, cols, rows, "bf16",
                               flags=flags, stream=on)
    sync()
    for t in (y, z, dx, dw):
        t.check_frame()
    want = ref.linear(a.numpy(), b.numpy(), bias.numpy()[0], "tanh", r.numpy(), "bf16")
    assert_within(y.numpy(), want[0], want[1], "y")
    assert_within(z.numpy(), want[2], want[3], "z")
    assert_within(dx.numpy(), *ref.product(a.numpy(), b.numpy(), "bf16", "swish",
                                           r.numpy()), "dx")
    assert_within(dw.numpy(), *ref.product(a.numpy(), b.numpy(), "bf16"), "dw")


@pytest.mark.parametrize("dtype,rows,cols,pad,shift", [
    ("f32", 1500, 1025, 0, 0), ("f32", 700, 2600, 1, 3), ("f32", 640, 4097, 2, 1),
    ("f32", 330, 5003, 0, 2), ("f32", 310, 8190, 1, 1), ("f32", 300, 9001, 0, 0),
    ("bf16", 1500, 1001, 0, 5), ("f16", 900, 2049, 2, 1), ("bf16", 620, 4097, 0, 7),
    ("bf16", 500, 5999, 4, 3), ("f16", 320, 8001, 0, 1), ("f64", 1300, 1025, 0, 1)])
def test_norms_of_many_rows_off_16_bytes(dtype, rows, cols, pad, shift):
    """Blocks that take several rows each, all cut at the same place, up to the
    tensor's last; the gradient in place of dy."""
    rng = np.random.default_rng(rows)
    x = inputs(rng, rows, cols, dtype, pad, shift, mean=2.0)
    dy = inputs(rng, rows, cols, dtype, pad, shift)
    g, b = inputs(rng, 1, cols, dtype), inputs(rng, 1, cols, dtype)
    wide = "f64" if dtype == "f64" else "f32"
    mean, rstd = Tensor(1, rows, wide), Tensor(1, rows, wide)
    y = Tensor(rows, cols, dtype, pad, shift)
    hx.cuda_layer_norm(0, x.ptr, y.ptr, rows, cols, dtype, gamma=g.ptr, beta=b.ptr,
                       mean=mean.ptr, rstd=rstd.ptr, ldx=x.ld, ldy=y.ld,
                       stream=stream())
    sync()
    y.check_frame()
    want = ref.layer_norm(x.numpy(), g.numpy()[0], b.numpy()[0], 1e-5, dtype)
    for got, (w, bound), what in ((y.numpy(), want[0], "y"),
                                  (mean.numpy()[0], want[1], "mean"),
                                  (rstd.numpy()[0], want[2], "rstd")):
        assert_within(got, w, bound, what)
    want = ref.layer_norm_grad(dy.numpy(), x.numpy(), mean.numpy()[0], rstd.numpy()[0],
                               g.numpy()[0], None, dtype)
    dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
    work = torch.empty(hx.grad_workspace_bytes(cols, dtype), device="cuda",
                       dtype=torch.uint8)
    hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, dy.ptr, rows, cols,
                            dtype, gamma=g.ptr, dgamma=dgamma.ptr, dbeta=dbeta.ptr,
                            workspace=work.data_ptr(), workspace_bytes=work.numel(),
                            lddy=dy.ld, ldx=x.ld, lddx=dy.ld, stream=stream())
    sync()
    dy.check_frame()
    assert_within(dy.numpy(), *want[0], "dx")
    assert_within(dgamma.numpy()[0], *want[1], "dgamma")
    assert_within(dbeta.numpy()[0], *want[2], "dbeta")


@pytest.mark.parametrize("flags", [0, GUARDED | _ffi.LINEAR_SPLIT(1),
                                   GUARDED | _ffi.LINEAR_SPLIT(4)])
@pytest.mark.parametrize("shift", [0, 1, 6])
def test_guarded_loads_at_the_ends_of_their_memory(flags, shift):
    """Operands that begin and end exactly where their buffers do (the first
    and last blocks reach outside them), at every phase of a row."""
    for m, n, k in ((129, 131, 193), (7, 9, 64), (130, 3, 129), (1, 1, 1)):
        rng = np.random.default_rng(m + shift)

        def exact(rows, cols):
            flat = torch.empty(shift + rows * cols, device="cuda", dtype=torch.bfloat16)
            t = flat[shift:].view(rows, cols)
            t.copy_(torch.as_tensor(normal(rng, (rows, cols))))
            return t
        x, w, wt, xt = exact(m, k), exact(k, n), exact(n, k), exact(k, m)
        outs = [Tensor(m, n, "bf16") for _ in range(3)]
        on = stream()
        hx.cuda_linear(0, x.data_ptr(), w.data_ptr(), outs[0].ptr, m, n, k, flags=flags,
                       stream=on)
        hx.cuda_linear_input_grad(0, x.data_ptr(), wt.data_ptr(), outs[1].ptr, m, k, n,
                                  flags=flags, stream=on)
        hx.cuda_linear_weight_grad(0, xt.data_ptr(), w.data_ptr(), outs[2].ptr, k, n, m,
                                   flags=flags, stream=on)
        sync()
        a = {id(t): t.double().cpu().numpy() for t in (x, w, wt, xt)}
        for out, left, right in ((outs[0], a[id(x)], a[id(w)]),
                                 (outs[1], a[id(x)], a[id(wt)].T),
                                 (outs[2], a[id(xt)].T, a[id(w)])):
            out.check_frame()
            assert_within(out.numpy(), *ref.product(left, right, "bf16"), "product")


# Rows whose tensors lie differently over 16 bytes, element by element: every
# length of such kernels, below its limit.
SINGLES = [("f32", 257, 0), ("f32", 1001, 0), ("f32", 511, 2), ("f32", 1500, 2),
           ("f32", 2049, 2), ("f32", 4095, 2), ("f32", 8000, 2), ("f64", 255, 0),
           ("f64", 511, 0), ("f64", 1025, 0), ("f64", 2047, 0), ("f64", 4095, 1)]


@pytest.mark.parametrize("dtype,cols,apart", SINGLES)
def test_gradients_of_single_elements_repeat(dtype, cols, apart):
    """The ring of rows of single elements: repeated with the inputs in turn in
    L2 and out of it, after NaNs have gone through the same shared memory, with
    and without dx and the residual, the gradients keep their bits, and they
    are right."""
    rng = np.random.default_rng(cols)
    rows, wide = 600, "f64" if dtype == "f64" else "f32"
    dy = inputs(rng, rows, cols, dtype, 1, 1)
    x = inputs(rng, rows, cols, dtype, 1, 1 + apart, 2.0, 1.0)
    residual = inputs(rng, rows, cols, dtype, 1, 1)
    gamma = inputs(rng, 1, cols, dtype, scale=0.2, mean=1.0)
    xd = x.numpy()
    mean = Tensor(1, rows, wide, data=xd.mean(1))
    rstd = Tensor(1, rows, wide, data=1 / np.sqrt(xd.var(1) + 1e-3))
    nans = Tensor(rows, cols + 1, dtype, data=np.full((rows, cols + 1), np.nan))
    nan_out = Tensor(rows, cols + 1, dtype, 0, 1)
    dx = Tensor(rows, cols, dtype, 1, 1)
    dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
    size = hx.grad_workspace_bytes(cols, dtype)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)
    flush = torch.empty(1 << 28, device="cuda", dtype=torch.uint8)
    first = {}
    for turn in range(24):
        if turn % 4 < 2:
            flush.fill_(turn)
        if turn % 3 == 0:   # leaves NaN in the ring's memory
            hx.cuda_layer_norm_grad(0, nans.ptr, nans.ptr, mean.ptr, rstd.ptr,
                                    nan_out.ptr, rows, cols + 1, dtype,
                                    residual=nans.ptr, stream=stream())
        form = turn % 2     # with all of dx and the residual, or the sums alone
        dx.view.fill_(FILL)
        hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr,
                                0 if form else dx.ptr, rows, cols, dtype,
                                gamma=gamma.ptr, dgamma=dgamma.ptr, dbeta=dbeta.ptr,
                                residual=0 if form else residual.ptr,
                                workspace=work.data_ptr(), workspace_bytes=size,
                                lddy=dy.ld, ldx=x.ld, lddx=dx.ld, ldr=residual.ld,
                                stream=stream())
        sync()
        got = [t.view.clone() for t in (dgamma, dbeta, dx)]
        for name, a, b in zip(("dgamma", "dbeta", "dx"), got,
                              first.setdefault(form, got)):
            assert torch.equal(a, b), f"{name}, turn {turn}"
    want = ref.layer_norm_grad(dy.numpy(), xd, mean.numpy()[0], rstd.numpy()[0],
                               gamma.numpy()[0], residual.numpy(), dtype)
    assert_within(first[0][2].double().cpu().numpy(), *want[0], "dx")
    for form in (0, 1):
        for (w, bound), got, what in zip(want[1:], first[form], ("dgamma", "dbeta")):
            assert_within(got.double().cpu().numpy()[0], w, bound, what)


LIMITS = {"none": (1, 1), "relu": (0, 1), "leaky_relu": (0.01, 1), "elu": (0, 1),
          "sigmoid": (0, 0), "tanh": (0, 0), "gelu": (0, 1), "swish": (0, 1),
          "mish": (0, 1)}


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_slopes_far_out_and_at_infinity_are_their_limits(act, dtype):
    """From |z| = 128 on every slope is its limit to f32 (e^-128 is below its
    smallest number), at the infinities too, where a type's largest value ends;
    a NaN stays one.  dy times 0, 1 or 0.01 is rounded once."""
    far = [128.0, 1e3, 1e4, 65504.0, float("inf")]
    z = torch.tensor([[-v for v in far] + far + [float("nan")]], device="cuda")
    z = z.repeat(40, 1).to(TORCH[dtype])
    dy = torch.randn(z.shape, device="cuda").to(TORCH[dtype])
    low, high = LIMITS[act]
    slopes = torch.tensor([low] * 5 + [high] * 5, device="cuda")
    want = (dy[:, :10].float() * slopes).to(TORCH[dtype])
    m, n = z.shape
    dz = torch.empty_like(dy)
    hx.cuda_linear_output_grad(0, dy.data_ptr(), m, n, dtype, act, preact=z.data_ptr(),
                               dz=dz.data_ptr(), stream=stream())
    # The same through a product: dx = (dy . 1) act'(z).
    one = torch.eye(n, device="cuda", dtype=TORCH[dtype])
    clean = torch.where(torch.isnan(z), torch.zeros_like(z), z)
    dx = torch.empty_like(dy)
    hx.cuda_linear_input_grad(0, dy.data_ptr(), one.data_ptr(), dx.data_ptr(), m, n, n,
                              dtype, act, preact=clean.data_ptr(), stream=stream())
    sync()
    assert bool((dz[:, :10] == want).all())
    assert bool((dx[:, :10] == want).all())
    assert bool(dx.isfinite().all())
    if act not in ("none", "relu", "leaky_relu"):
        assert bool(dz[:, 10].isnan().all())


@pytest.mark.parametrize("act", ["gelu", "swish", "mish"])
def test_preactivations_beyond_f16_have_finite_gradients(act):
    """z = -102400 and 102400: y has its value (0, or beyond f16), z is stored
    as an infinity, and the slope there is 0 or 1."""
    m, n, k = 20, 16, 64
    x = torch.full((m, k), 40.0, device="cuda", dtype=torch.float16)
    w = torch.full((k, n), 40.0, device="cuda", dtype=torch.float16)
    w[:, ::2] = -40.0
    y, z, dz = (torch.empty(m, n, device="cuda", dtype=torch.float16) for _ in range(3))
    dy = torch.randn(m, n, device="cuda").half()
    db = torch.empty(n, device="cuda", dtype=torch.float16)
    work = torch.empty(hx.grad_workspace_bytes(n, "f16"), device="cuda",
                       dtype=torch.uint8)
    hx.cuda_linear(0, x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k, "f16", act,
                   preact=z.data_ptr(), stream=stream())
    hx.cuda_linear_output_grad(0, dy.data_ptr(), m, n, "f16", act, preact=z.data_ptr(),
                               dz=dz.data_ptr(), dbias=db.data_ptr(),
                               workspace=work.data_ptr(), workspace_bytes=work.numel(),
                               stream=stream())
    sync()
    assert bool((y[:, ::2] == 0).all()) and bool(z.isinf().all())
    assert bool((dz[:, ::2] == 0).all()) and bool((dz[:, 1::2] == dy[:, 1::2]).all())
    assert bool(db.isfinite().all())


@pytest.mark.parametrize("act", ref.ACTS)
def test_activations_of_large_finite_sums(act):
    """act(z) for z far beyond the fitted range of the normal distribution's
    polynomial: to f32's precision z or its limit, so y has the rounded value."""
    zs = torch.tensor([14.0, 14.5, 20.0, 40.0, 90.0, 128.0, 1e3, 1e10, 3e38],
                      device="cuda")
    zs = torch.cat([-zs, zs]).bfloat16()
    n = zs.numel()
    x = torch.ones(3, 1, device="cuda", dtype=torch.bfloat16)
    y = torch.empty(3, n, device="cuda", dtype=torch.bfloat16)
    hx.cuda_linear(0, x.data_ptr(), zs.data_ptr(), y.data_ptr(), 3, n, 1, "bf16", act,
                   stream=stream())
    sync()
    z = zs.double().cpu().numpy()
    want = np.where(z > 0, z, 0.0) if act in ("gelu", "swish", "mish") else ref.act(act, z)
    if act in ("swish", "mish"):   # z e^z below, above z within its rounding
        want = np.where(z < 0, z * np.exp(z.clip(-700, 0)), z)
    # Below -87 exponentials are subnormal in f32: 2^-149 of absolute error,
    # times z.  gelu at -14 is below 1e-43, the subnormals' last digits.
    bound = np.abs(want) * (ref.HALF["bf16"] * 2 + (16 + 4 * np.abs(z).clip(0, 200))
                            * ref.U32) + 2.0 ** -133 + 2.0 ** -149 * np.abs(z).clip(0, 128)
    if act == "gelu":
        bound = bound + 1e-43
    for row in y.double().cpu().numpy():
        assert_within(row, want, bound, act)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("cols,pad", [(1, 0), (1, 1), (2, 0), (3, 0), (5, 1), (7, 0),
                                      (8, 1)])
def test_norms_of_rows_shorter_than_16_bytes(dtype, cols, pad):
    """Several rows share a 16-byte block, at every offset of the tensor into
    one; what lies around the tensors is NaN and does not reach the results."""
    rows, per = 41, 16 // torch.empty(0, dtype=TORCH[dtype]).element_size()
    wide = "f64" if dtype == "f64" else "f32"
    rng = np.random.default_rng(cols)
    for shift in range(per):
        x, dy = (inputs(rng, rows, cols, dtype, pad, shift) for _ in range(2))
        for t in (x, dy):
            t.flat[:t.start] = float("nan")
            t.flat[t.start + (rows - 1) * t.ld + cols:] = float("nan")
        y, dx = (Tensor(rows, cols, dtype, pad, shift) for _ in range(2))
        mean, rstd = Tensor(1, rows, wide), Tensor(1, rows, wide)
        dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
        size = hx.grad_workspace_bytes(cols, dtype)
        work = torch.empty(size, device="cuda", dtype=torch.uint8)
        hx.cuda_layer_norm(0, x.ptr, y.ptr, rows, cols, dtype, mean=mean.ptr,
                           rstd=rstd.ptr, eps=0.5, ldx=x.ld, ldy=y.ld, stream=stream())
        hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, dx.ptr, rows,
                                cols, dtype, dgamma=dgamma.ptr, dbeta=dbeta.ptr,
                                workspace=work.data_ptr(), workspace_bytes=size,
                                lddy=dy.ld, ldx=x.ld, lddx=dx.ld, stream=stream())
        sync()
        for t in (y, dx):
            t.check_frame()
        (want, bound), _, _ = ref.layer_norm(x.numpy(), None, None, 0.5, dtype)
        assert_within(y.numpy(), want, bound, f"y, shift {shift}")
        want = ref.layer_norm_grad(dy.numpy(), x.numpy(), mean.numpy()[0],
                                   rstd.numpy()[0], None, None, dtype)
        for got, (w, bound), what in ((dx.numpy(), want[0], "dx"),
                                      (dgamma.numpy()[0], want[1], "dgamma"),
                                      (dbeta.numpy()[0], want[2], "dbeta")):
            assert_within(got, w, bound, f"{what}, shift {shift}")


PLANNED = [("forward", 136, 5960, 8), ("forward", 300, 520, 1000), ("forward", 48, 512, 512),
           ("forward", 777, 1001, 153), ("input_grad", 280, 8, 3416),
           ("input_grad", 300, 520, 1000), ("weight_grad", 8, 4832, 144),
           ("weight_grad", 513, 72, 2056)]


@pytest.mark.parametrize("op,m,n,k", PLANNED)
def test_the_plan_is_what_runs(op, m, n, k):
    """The kernel a call would launch (an injected launch fault names it),
    against linear_plan for the same facts: with and without what the epilogue
    reads, with each tensor on 16-byte rows and off them."""
    names = {1: "pair", 2: "single", 3: "skinny", 4: "guarded"}
    shapes = {"forward": ((m, k), (k, n), (m, n)),
              "input_grad": ((m, n), (k, n), (m, k)),
              "weight_grad": ((m, k), (m, n), (k, n))}[op]

    def tensor(shape, aligned):
        rows, cols = shape
        ld = -(-cols // 8) * 8 + (0 if aligned else 1)
        return torch.zeros(rows, ld, device="cuda", dtype=torch.bfloat16)
    for aligned in (14, 2, 4, 6, 12, 0):
        a, b, out = (tensor(s, aligned >> 1 + i & 1) for i, s in enumerate(shapes))
        for reads in (False, True):
            if reads and op == "weight_grad":
                continue
            args = (0, a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k)
            r = out.data_ptr() if reads else 0
            la, lb, lo = a.stride(0), b.stride(0), out.stride(0)
            hx.fault_configure("launch:1")
            try:
                with pytest.raises(_ffi.HexirError) as err:
                    if op == "forward":
                        hx.cuda_linear(*args, residual=r, ldx=la, ldw=lb, ldy=lo,
                                       ldr=lo, stream=stream())
                    elif op == "input_grad":
                        hx.cuda_linear_input_grad(*args, residual=r, lddz=la, ldw=lb,
                                                  lddx=lo, ldr=lo, stream=stream())
                    else:
                        hx.cuda_linear_weight_grad(*args, ldx=la, lddz=lb, lddw=lo,
                                                   stream=stream())
            finally:
                hx.fault_configure("")
            plan = hx.linear_plan(op, m, n, k, aligned, plain=not reads)
            assert f"hexir_linear_16 {names[plan[0]]}:" in str(err.value), \
                (aligned, reads, plan, str(err.value))


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(3, 7), (3000, 40), (2500, 256), (1500, 1000),
                                       (1300, 1024), (700, 1025), (700, 3001),
                                       (330, 4096), (330, 5000), (170, 8192),
                                       (170, 16384), (5, 16385)])
def test_norms_of_tensors_that_lie_differently(dtype, rows, cols):
    """Every tensor has an alignment and a stride of its own, so that rows go
    element by element in every type, at the lengths where the kernels change;
    several rows a block; the gradient also in place of the residual."""
    rng = np.random.default_rng(rows + cols)
    wide = "f64" if dtype == "f64" else "f32"
    x = inputs(rng, rows, cols, dtype, 1, 1, 2.0, 1.0)
    y = Tensor(rows, cols, dtype, 0, 2)
    dy = inputs(rng, rows, cols, dtype, 2, 3)
    residual = inputs(rng, rows, cols, dtype, 5, 2)
    dx = Tensor(rows, cols, dtype, 16, 0)
    gamma = inputs(rng, 1, cols, dtype, shift=1, scale=0.2, mean=1.0)
    beta = inputs(rng, 1, cols, dtype, shift=3, scale=0.2)
    mean, rstd = Tensor(1, rows, wide, shift=1), Tensor(1, rows, wide)
    dgamma, dbeta = Tensor(1, cols, dtype, shift=1), Tensor(1, cols, dtype, shift=2)
    size = hx.grad_workspace_bytes(cols, dtype)
    work = torch.full((size + 64,), 0xA5, device="cuda", dtype=torch.uint8)
    hx.cuda_layer_norm(0, x.ptr, y.ptr, rows, cols, dtype, gamma=gamma.ptr,
                       beta=beta.ptr, mean=mean.ptr, rstd=rstd.ptr, eps=1e-5, ldx=x.ld,
                       ldy=y.ld, stream=stream())
    sync()
    want = ref.layer_norm(x.numpy(), gamma.numpy()[0], beta.numpy()[0], 1e-5, dtype)
    for t, (w, bound), what in ((y, want[0], "y"), (mean, want[1], "mean"),
                                (rstd, want[2], "rstd")):
        t.check_frame()
        got = t.numpy()
        assert_within(got if what == "y" else got[0], w, bound, what)
    want = ref.layer_norm_grad(dy.numpy(), x.numpy(), mean.numpy()[0], rstd.numpy()[0],
                               gamma.numpy()[0], residual.numpy(), dtype)
    for out in (dx, residual):
        hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, out.ptr, rows,
                                cols, dtype, gamma=gamma.ptr, dgamma=dgamma.ptr,
                                dbeta=dbeta.ptr, residual=residual.ptr,
                                workspace=work.data_ptr(), workspace_bytes=size,
                                lddy=dy.ld, ldx=x.ld, lddx=out.ld, ldr=residual.ld,
                                stream=stream())
        sync()
        assert bool((work[size:] == 0xA5).all()), "a write behind the workspace"
        for t, (w, bound), what in ((out, want[0], "dx"), (dgamma, want[1], "dgamma"),
                                    (dbeta, want[2], "dbeta")):
            t.check_frame()
            got = t.numpy()
            assert_within(got if what == "dx" else got[0], w, bound, what)


def run_fresh(body):
    """`body` in a process of its own, whose device code is not loaded yet."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    head = ("import torch\nimport hexir_b200 as hx\n"
            "from tests.test_gpu_layers import Block, feed_forward, sync, stream\n")
    done = subprocess.run([sys.executable, "-c", head + body], cwd=root, timeout=300,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


def test_an_empty_call_is_enough_before_a_capture():
    """In a new process: one empty call, then a step whose kernels have never run
    is captured, behind copies (nodes that are no kernels), and replayed."""
    run_fresh("""
hx.cuda_linear(0, 0, 0, 0, 0, 8, 8)
shapes = [(260, 256, 1000), (3, 130, 515), (40, 1024, 4096)]
blocks = [(Block(*s), feed_forward(*s, seed=1), feed_forward(*s, seed=2)) for s in shapes]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    on = torch.cuda.current_stream().cuda_stream
    for block, p, fresh in blocks:
        for k in p:
            p[k].copy_(fresh[k])
        block.forward(p, on)
        block.backward(p, on)
graph.replay()
sync()
for (block, p, fresh), s in zip(blocks, shapes):
    other = Block(*s)
    other.forward(fresh, stream())
    other.backward(fresh, stream())
    sync()
    for (name, a), b in zip(block.outputs().items(), other.outputs().values()):
        assert torch.equal(a, b), (s, name)
""")


@pytest.mark.parametrize("dtype,size", [("bf16", 120), ("f32", 120), ("f64", 1016)])
@pytest.mark.parametrize("cols,pad,shift", [(64, 0, 0), (40, 0, 0), (41, 0, 3), (41, 3, 1),
                                            (100, 0, 0)])
def test_gradient_of_constant_rows_of_large_numbers(dtype, size, cols, pad, shift):
    """x - mean is 0 and xhat with it, although mean * rstd is beyond the type's
    range: threads without an element of the row must not bring it in.  Results
    and bounds are those of x = mean = 0, whose xhat is as exact."""
    wide, rows = "f64" if dtype == "f64" else "f32", 30
    rng = np.random.default_rng(cols)
    x = Tensor(rows, cols, dtype, pad, shift, np.full((rows, cols), 2.0 ** size))
    x.view[::2] *= -1
    dy = inputs(rng, rows, cols, dtype, pad, shift)
    mean = Tensor(1, rows, wide, data=x.numpy()[:, 0])
    rstd = Tensor(1, rows, wide, data=np.full(rows, 512.0))
    dx = Tensor(rows, cols, dtype, pad, shift)
    dgamma, dbeta = Tensor(1, cols, dtype), Tensor(1, cols, dtype)
    work = torch.empty(hx.grad_workspace_bytes(cols, dtype), device="cuda",
                       dtype=torch.uint8)
    hx.cuda_layer_norm_grad(0, dy.ptr, x.ptr, mean.ptr, rstd.ptr, dx.ptr, rows, cols,
                            dtype, dgamma=dgamma.ptr, dbeta=dbeta.ptr,
                            workspace=work.data_ptr(), workspace_bytes=work.numel(),
                            lddy=dy.ld, ldx=x.ld, lddx=dx.ld, stream=stream())
    sync()
    want = ref.layer_norm_grad(dy.numpy(), np.zeros((rows, cols)), np.zeros(rows),
                               rstd.numpy()[0], None, None, dtype)
    assert_within(dx.numpy(), *want[0], "dx")
    assert_within(dgamma.numpy()[0], *want[1], "dgamma")
    assert_within(dbeta.numpy()[0], *want[2], "dbeta")


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 1, 9), (5, 9, 1), (63, 1001, 77),
                                   (129, 7, 513), (200, 249, 129), (300, 515, 67)])
@pytest.mark.parametrize("dtype,extra", [("bf16", 0), ("f16", 8)])
def test_odd_extents_on_16_byte_rows_in_every_kernel(m, n, k, dtype, extra):
    """Rows of any length inside buffers whose rows start on 16-byte (and, by
    `extra`, not on 32-byte) boundaries: what lies in the gaps is NaN."""
    rng = np.random.default_rng(m + n + k)

    def padded(rows, cols, data=None):
        t = Tensor(rows, cols, dtype, -cols % 8 + extra,
                   data=normal(rng, (rows, cols)) if data is None else data)
        keep = t.view.clone()
        t.flat.fill_(float("nan"))
        t.view.copy_(keep)
        return t
    x, w, wt = padded(m, k), padded(k, n), padded(n, k)
    xt, r, z0 = padded(k, m), padded(m, n), padded(m, n)
    on = stream()
    flags = [0, GUARDED | _ffi.LINEAR_SPLIT(2), SINGLE | _ffi.LINEAR_SPLIT(1),
             SINGLE | _ffi.LINEAR_TILE(64) | _ffi.LINEAR_SPLIT(4),
             PAIR | _ffi.LINEAR_TILE(128), PAIR | _ffi.LINEAR_TILE(256)]
    for flag in flags + ([SKINNY, SKINNY | _ffi.LINEAR_SPLIT(4)] if m <= 64 else []):
        y, z, dx, dw = (Tensor(m, n, dtype, -n % 8 + extra) for _ in range(4))
        hx.cuda_linear(0, x.ptr, w.ptr, y.ptr, m, n, k, dtype, "gelu",
                       bias=r.ptr, residual=r.ptr, preact=z.ptr, ldx=x.ld, ldw=w.ld,
                       ldy=y.ld, ldr=r.ld, ldp=z.ld, flags=flag, stream=on)
        if not flag & SKINNY:
            hx.cuda_linear_input_grad(0, x.ptr, wt.ptr, dx.ptr, m, k, n, dtype, "swish",
                                      preact=z0.ptr, residual=r.ptr, lddz=x.ld,
                                      ldw=wt.ld, lddx=dx.ld, ldp=z0.ld, ldr=r.ld,
                                      flags=flag, stream=on)
            hx.cuda_linear_weight_grad(0, xt.ptr, w.ptr, dw.ptr, k, n, m, dtype,
                                       ldx=xt.ld, lddz=w.ld, lddw=dw.ld, flags=flag,
                                       stream=on)
        sync()
        for t in (y, z, dx, dw):
            t.check_frame()
        want = ref.linear(x.numpy(), w.numpy(), r.numpy()[0], "gelu", r.numpy(), dtype)
        assert_within(y.numpy(), want[0], want[1], f"y {flag:#x}")
        assert_within(z.numpy(), want[2], want[3], f"z {flag:#x}")
        if not flag & SKINNY:
            assert_within(dx.numpy(), *ref.product(
                x.numpy(), wt.numpy().T, dtype, "swish", z0.numpy(), r.numpy()),
                f"dx {flag:#x}")
            assert_within(dw.numpy(), *ref.product(xt.numpy().T, w.numpy(), dtype),
                          f"dw {flag:#x}")


def test_layers_through_the_packages_own_buffers_and_streams():
    """Without torch: the framework's device buffers, on the device's stream."""
    rows, cols = 37, 64
    rng = np.random.default_rng(5)
    dev = hx.Device("cuda")
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    bx, by = dev.buffer(x.nbytes), dev.buffer(x.nbytes)
    bx.write(x)
    hx.cuda_layer_norm(0, bx.ptr, by.ptr, rows, cols, "f32", eps=1e-5, stream=dev.stream)
    hx.cuda_synchronize(0, dev.stream)
    (want, bound), _, _ = ref.layer_norm(x.astype(np.float64), None, None, 1e-5, "f32")
    assert_within(by.read((rows, cols), np.float32).astype(np.float64), want, bound, "y")


@pytest.mark.parametrize("rows,cols", [(150, 131), (700, 259), (131, 1027)])
def test_calls_back_to_back_read_what_the_call_before_wrote(rows, cols):
    """A chain of calls that read each other's outputs, off 16 bytes and in
    buffers that every pass writes anew (so that an old line of a cache would
    show), queued without a pause, against the same chain with a pause after each
    call."""
    rng = np.random.default_rng(rows)
    start = normal(rng, (rows, cols))
    w = inputs(rng, cols, cols, "bf16", 1, 1, scale=cols ** -0.5)

    def chain(pause):
        a, b = (Tensor(rows, cols, "bf16", 1, 1, start) for _ in range(2))
        dw = Tensor(cols, cols, "bf16", 1, 1)
        dbias = Tensor(1, cols, "bf16")
        work = torch.empty(hx.grad_workspace_bytes(cols), device="cuda",
                           dtype=torch.uint8)
        on = stream()
        seen = []
        for _ in range(12):
            for call in (
                    lambda: hx.cuda_linear(0, a.ptr, w.ptr, b.ptr, rows, cols, cols,
                                           residual=b.ptr, ldx=a.ld, ldw=w.ld, ldy=b.ld,
                                           ldr=b.ld, stream=on),
                    lambda: hx.cuda_layer_norm(0, b.ptr, a.ptr, rows, cols, "bf16",
                                               ldx=b.ld, ldy=a.ld, stream=on),
                    lambda: hx.cuda_linear_weight_grad(0, a.ptr, b.ptr, dw.ptr, rows,
                                                       cols, cols, ldx=a.ld, lddz=b.ld,
                                                       lddw=dw.ld, stream=on),
                    lambda: hx.cuda_linear_input_grad(0, b.ptr, w.ptr, a.ptr, rows, cols,
                                                      cols, residual=a.ptr, lddz=b.ld,
                                                      ldw=w.ld, lddx=a.ld, ldr=a.ld,
                                                      stream=on),
                    lambda: hx.cuda_linear_output_grad(0, a.ptr, rows, cols, "bf16",
                                                       "swish", preact=b.ptr, dz=a.ptr,
                                                       dbias=dbias.ptr,
                                                       workspace=work.data_ptr(),
                                                       workspace_bytes=work.numel(),
                                                       lddy=a.ld, ldp=b.ld, lddz=a.ld,
                                                       stream=on),
                    lambda: hx.cuda_layer_norm(0, a.ptr, a.ptr, rows, cols, "bf16",
                                               ldx=a.ld, ldy=a.ld, stream=on)):
                call()
                if pause:
                    sync()
            seen.append([t.view.clone() for t in (a, b, dw, dbias)])
        sync()
        return seen
    want = chain(True)
    for _ in range(10):
        for i, (got, expected) in enumerate(zip(chain(False), want)):
            for name, g, e in zip(("a", "b", "dw", "dbias"), got, expected):
                assert torch.equal(g, e), (i, name)
