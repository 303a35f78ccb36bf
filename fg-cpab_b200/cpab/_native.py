"""ctypes binding of libcpab_b200.so (the C ABI in include/cpab_b200.h).

Tensors cross the boundary as raw device pointers plus sizes; every call is
enqueued on torch's current stream of the tensors' device.  There is no CPU
fallback: if the library is missing or the tensors are not CUDA tensors the
call raises.
"""
import contextlib
import ctypes
import functools
import os

import torch

# The library built next to this file; CPAB_B200_LIB names another build of
# the same ABI (e.g. one with other compile-time kernel choices).
LIB_PATH = os.environ.get("CPAB_B200_LIB") or os.path.join(
    os.path.dirname(os.path.abspath(__file__)), "libcpab_b200.so")

_c_int, _c_i64, _c_float, _p = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

# name -> argtypes (all return int status)
_SIGNATURES = {
    "cpab_b200_expm": [_c_int, _p, _c_i64, _c_float, _p, _p],
    "cpab_b200_build_A": [_c_int, _c_i64, _c_i64, _c_int, _p, _p, _p, _p, _c_float, _p, _p, _p],
    "cpab_b200_forward": [_c_int, _p, _p, _c_i64, _c_int, _p, _p, _p, _c_int, _c_int, _c_int, _p,
                          _p],
    "cpab_b200_forward_1d_closed_form": [_p, _c_i64, _c_int, _p, _p, _c_int, _c_int, _p, _p],
    "cpab_b200_backward": [_c_int, _p, _p, _c_i64, _c_int, _p, _p, _c_int, _p, _c_int, _c_int,
                           _p, _p, _p],
    "cpab_b200_order_points": [_c_int, _p, _p, _c_i64, _c_int, _p, _p, _p],
    "cpab_b200_order_points_static": [_c_int, _p, _p, _c_i64, _c_int, _p, _p],
    "cpab_b200_cell_index": [_c_int, _p, _p, _c_i64, _p, _p],
    "cpab_b200_project": [_c_i64, _c_i64, _c_int, _p, _p, _p, _p, _p, _p],
    "cpab_b200_build_A_tt": [_c_int, _c_i64, _c_i64, _c_int, _p, _p, _p, _p, _c_float, _p, _p, _p],
    "cpab_b200_project_tt": [_c_i64, _c_i64, _c_int, _p, _p, _p, _p, _p, _p],
    "cpab_b200_interpolate": [_c_int, _p, _c_int, _c_int, _p, _p, _p, _p, _p],
    "cpab_b200_interpolate_backward": [_c_int, _p, _c_int, _c_int, _p, _p, _p, _p, _p, _p, _p],
    "cpab_b200_forward_chain": [_c_int, _p, _p, _c_i64, _c_int, _p, _p, _p, _c_int, _c_int,
                                _c_int, _c_int, _p, _p, _p],
    "cpab_b200_backward_chain": [_c_int, _p, _p, _c_i64, _c_int, _p, _p, _c_int, _c_int, _p, _p,
                                 _c_int, _c_int, _p, _p, _p],
    "cpab_b200_transform_data": [_c_int, _p, _p, _p, _p, _p, _p, _c_int, _c_int, _c_int, _p,
                                 _c_int, _p, _p, _p, _p],
    "cpab_b200_transform_data_backward": [_c_int, _p, _p, _p, _p, _p, _c_int, _c_int, _c_int,
                                          _p, _c_int, _p, _p, _p, _p, _p, _p],
    "cpab_b200_warp": [_c_int, _p, _p, _p, _p, _p, _p, _c_int, _c_int, _c_int, _c_int, _p,
                       _c_int, _c_int, _p, _c_int, _p, _p, _p, _p],
    "cpab_b200_warp_backward": [_c_int, _p, _p, _p, _p, _p, _c_int, _c_int, _c_int, _c_int, _p,
                                _c_int, _c_int, _p, _c_int, _p, _p, _p, _p, _p, _p],
    "cpab_b200_gated_scan": [_c_int, _p, _c_i64, _c_i64, _p, _c_i64, _c_i64, _c_i64, _c_i64,
                             _c_i64, _p, _p, _p, _p, _p, _p, _p],
    "cpab_b200_gated_scan_backward": [_c_int, _p, _c_i64, _c_i64, _p, _c_i64, _c_i64, _c_i64,
                                      _c_i64, _c_i64, _p, _p, _p, _p, _p, _c_i64, _c_i64, _p,
                                      _c_i64, _c_i64, _p, _p, _p],
    "cpab_b200_gated_scan_step": [_c_int, _p, _c_i64, _p, _c_i64, _c_i64, _c_i64, _p, _c_i64, _p,
                                  _p, _p],
    "cpab_b200_rms_norm": [_c_int, _c_int, _c_int, _p, _c_i64, _p, _c_i64, _p, _c_i64, _c_i64,
                           _c_float, _p, _p, _p, _p],
    "cpab_b200_rms_norm_quantized": [_c_int, _c_int, _c_int, _p, _c_i64, _p, _c_i64, _p, _c_i64,
                                     _c_i64, _c_float, _p, _p, _p, _p],
    "cpab_b200_rms_norm_backward": [_c_int, _c_int, _c_int, _p, _c_i64, _p, _p, _c_i64, _c_i64,
                                    _p, _p, _p, _p, _p, _p, _p],
    "cpab_b200_adamw": [_p, _c_int, ctypes.c_uint32, _p, _p],
    "cpab_b200_quantize_blocks": [_c_int, _p, _c_i64, _c_i64, _c_i64, _p, _c_i64, _p, _c_i64, _p,
                                  _c_i64, _p, _c_i64, _c_int, _p, _p, _p],
    "cpab_b200_matmul_quantized": [_c_int, _p, _p, _c_i64, _c_i64, _c_i64, _c_int, _p, _p, _c_i64,
                                   _p, _p],
    "cpab_b200_set_wait_limit": [_c_i64],
    "cpab_b200_lay_out_codes": [_c_int, _p, _p, _p, _p, _c_i64, _p],
    "cpab_b200_orthogonalize": [_c_int, _p, _c_i64, _c_i64, _c_i64, _c_int, _p, ctypes.c_double, _p,
                                _p, _p],
    "cpab_b200_muon": [_p, _c_int, ctypes.c_double, _p, ctypes.c_double, _c_int, ctypes.c_double,
                       _c_int, _p, ctypes.c_double, _c_int, _p, _p],
}

# Entry points that return something else than a status.
_OTHERS = {
    "cpab_b200_version": (ctypes.c_int, []),
    "cpab_b200_max_steps": (ctypes.c_int, []),
    "cpab_b200_last_error": (ctypes.c_char_p, []),
    "cpab_b200_gated_scan_chunk": (ctypes.c_int, []),
    "cpab_b200_gated_scan_workspace": (_c_i64, [_c_int, _c_i64, _c_i64, _c_i64]),
    "cpab_b200_rms_norm_workspace": (_c_i64, [_c_int, _c_i64, _c_i64]),
    "cpab_b200_quantize_blocks_workspace": (_c_i64, [_c_i64, _c_i64]),
    "cpab_b200_matmul_quantized_workspace": (_c_i64, [_c_i64, _c_i64, _c_i64]),
    "cpab_b200_orthogonalize_workspace": (_c_i64, [_c_int, _c_i64, _c_i64, _c_i64]),
    "cpab_b200_muon_workspace": (_c_i64, [_p, _c_int]),
}

EXPORTS = tuple(_SIGNATURES) + tuple(_OTHERS)

_lib = None


class CpabNativeError(RuntimeError):
    """A libcpab_b200 call returned a non-zero status."""


def lib():
    """Load (once) and return the native library."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                "libcpab_b200.so is not built (expected at %s); run "
                "`python fg-cpab_b200/build.py` first" % LIB_PATH)
        L = ctypes.CDLL(LIB_PATH)
        for name, args in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = ctypes.c_int
        for name, (res, args) in _OTHERS.items():
            getattr(L, name).restype = res
            getattr(L, name).argtypes = args
        _lib = L
    return _lib


def max_steps():
    return lib().cpab_b200_max_steps()


def _check(status):
    if status != 0:
        msg = lib().cpab_b200_last_error().decode(errors="replace")
        raise CpabNativeError(msg or "libcpab_b200 error %d" % status)


def _ptr(t):
    """Device pointer of t (None = NULL); ctypes converts it for the void* arguments."""
    return t.data_ptr() if t is not None else None


# The raw cudaStream_t of the current stream in one call (torch's own query for
# generated kernels); current_stream() builds a Stream object per call, which
# is a sizeable share of a call's host time.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    index = device.index if device.index is not None else torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(device).cuda_stream


def _require(t, name, dtype=torch.float32):
    if not t.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor (no CPU path)" % name)
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if not t.is_contiguous():
        raise RuntimeError("%s must be contiguous" % name)


@functools.lru_cache(maxsize=256)
def _i32_cached(values):
    return (ctypes.c_int32 * len(values))(*values)


@functools.lru_cache(maxsize=256)
def _i64_cached(values):
    return (ctypes.c_int64 * len(values))(*values)


def _i32_array(values):
    """Read-only int32 array for a call (tessellation sizes): cached per value."""
    return _i32_cached(tuple(int(v) for v in values))


def _i64_array(values):
    """Read-only int64 array for a call (tensor sizes): cached per value."""
    return _i64_cached(tuple(int(v) for v in values))


def _on(device):
    """Context making `device` current; nothing to do when it already is."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


# ---------------------------------------------------------------------------
# Thin wrappers: shapes in, tensors out (allocated with torch on the device).
# ---------------------------------------------------------------------------

def expm(As, dT):
    """Trels = expm(dT * A) for As [n, ndim, ndim+1]."""
    _require(As, "As")
    n, nd = As.shape[0], As.shape[1]
    out = torch.empty_like(As)
    with _on(As.device):
        _check(lib().cpab_b200_expm(nd, _ptr(As), n, float(dT), _ptr(out), _stream(As.device)))
    return out


def build_A(ndim, nC, basis, theta, dT=None):
    """As = reshape(B theta^T) [n_theta, nC, ndim, ndim+1] and, when dT is given,
    Trels = expm(dT * As).  ``basis`` is a DeviceBasis."""
    _require(theta, "theta")
    n_theta = theta.shape[0]
    As = torch.empty((n_theta, nC, ndim, ndim + 1), device=theta.device, dtype=torch.float32)
    trels = torch.empty_like(As) if dT is not None else None
    with _on(theta.device):
        _check(lib().cpab_b200_build_A(
            ndim, nC, basis.d, n_theta, _ptr(basis.rowptr), _ptr(basis.colidx), _ptr(basis.vals),
            _ptr(theta), float(dT) if dT is not None else 0.0, _ptr(As), _ptr(trels),
            _stream(theta.device)))
    return As, trels


def build_A_tt(ndim, nC, basis, theta_t, n_theta, dT=None):
    """build_A with theta given transposed, theta_t [d, n_theta]."""
    _require(theta_t, "theta_t")
    As = torch.empty((n_theta, nC, ndim, ndim + 1), device=theta_t.device, dtype=torch.float32)
    trels = torch.empty_like(As) if dT is not None else None
    with _on(theta_t.device):
        _check(lib().cpab_b200_build_A_tt(
            ndim, nC, basis.d, n_theta, _ptr(basis.rowptr), _ptr(basis.colidx), _ptr(basis.vals),
            _ptr(theta_t), float(dT) if dT is not None else 0.0, _ptr(As), _ptr(trels),
            _stream(theta_t.device)))
    return As, trels


def order_points(nc, points, batched):
    """Processing order of the points sorted by initial cell: int32
    [n_sets, nP] (n_sets = batch when batched, else 1)."""
    _require(points, "points")
    nd, nP = points.shape[-2], points.shape[-1]
    n_sets = points.shape[0] if batched else 1
    nC = int(np_prod(nc)) * {1: 1, 2: 4, 3: 5}[nd]
    counts = torch.empty((n_sets, nC), device=points.device, dtype=torch.int32)
    order = torch.empty((n_sets, nP), device=points.device, dtype=torch.int32)
    with _on(points.device):
        _check(lib().cpab_b200_order_points(nd, _i32_array(nc), _ptr(points), nP, n_sets,
                                            _ptr(counts), _ptr(order), _stream(points.device)))
    return order


def np_prod(xs):
    r = 1
    for x in xs:
        r *= int(x)
    return r


def forward(ndim, nc, points, batched, trels, As, nstepsolver, adaptive, order=None):
    _require(points, "points")
    _require(As, "As")
    n_theta = As.shape[0]
    nP = points.shape[-1]
    out = torch.empty((n_theta, ndim, nP), device=As.device, dtype=torch.float32)
    with _on(As.device):
        if ndim == 1:
            _check(lib().cpab_b200_forward_1d_closed_form(
                _ptr(points), nP, int(batched), _ptr(order), _ptr(As), n_theta, int(nc[0]),
                _ptr(out), _stream(As.device)))
        else:
            _require(trels, "Trels")
            _check(lib().cpab_b200_forward(
                ndim, _i32_array(nc), _ptr(points), nP, int(batched), _ptr(order), _ptr(trels),
                _ptr(As), n_theta, int(nstepsolver), int(adaptive), _ptr(out),
                _stream(As.device)))
    return out


def backward(ndim, nc, points, batched, As, grad_out, nstepsolver, adaptive, want_points,
             order=None):
    """Returns (moments [n_theta, nC, ppc], grad_points [n_theta, ndim, nP] or None)."""
    _require(points, "points")
    _require(As, "As")
    _require(grad_out, "grad")
    n_theta, nC = As.shape[0], As.shape[1]
    nP = points.shape[-1]
    ppc = ndim * (ndim + 1)
    moments = torch.empty((n_theta, nC, ppc), device=As.device, dtype=torch.float32)
    gp = (torch.empty((n_theta, ndim, nP), device=As.device, dtype=torch.float32)
          if want_points else None)
    with _on(As.device):
        _check(lib().cpab_b200_backward(
            ndim, _i32_array(nc), _ptr(points), nP, int(batched), _ptr(order), _ptr(As), n_theta,
            _ptr(grad_out), int(nstepsolver), int(adaptive), _ptr(moments), _ptr(gp),
            _stream(As.device)))
    return moments, gp


def cell_index(nc, points):
    """Cell of every point, points [ndim, n] -> int32 [n]."""
    _require(points, "points")
    nd, n = points.shape
    out = torch.empty(n, device=points.device, dtype=torch.int32)
    with _on(points.device):
        _check(lib().cpab_b200_cell_index(nd, _i32_array(nc), _ptr(points), n, _ptr(out),
                                          _stream(points.device)))
    return out


def project(basis, moments):
    """dtheta [n_theta, d] = B^T vec(moments)."""
    _require(moments, "moments")
    n_theta = moments.shape[0]
    D = moments[0].numel()
    out = torch.empty((n_theta, basis.d), device=moments.device, dtype=torch.float32)
    with _on(moments.device):
        _check(lib().cpab_b200_project(
            basis.d, D, n_theta, _ptr(basis.t_rowptr), _ptr(basis.t_colidx), _ptr(basis.t_vals),
            _ptr(moments), _ptr(out), _stream(moments.device)))
    return out


def project_tt(basis, moments_t, n_theta):
    """project with the moments given transposed, moments_t [D, n_theta]."""
    _require(moments_t, "moments_t")
    out = torch.empty((n_theta, basis.d), device=moments_t.device, dtype=torch.float32)
    with _on(moments_t.device):
        _check(lib().cpab_b200_project_tt(
            basis.d, moments_t.shape[0], n_theta, _ptr(basis.t_rowptr), _ptr(basis.t_colidx),
            _ptr(basis.t_vals), _ptr(moments_t), _ptr(out), _stream(moments_t.device)))
    return out


def interpolate(ndim, data, grid, outsize):
    _require(data, "data")
    _require(grid, "grid")
    B, C = data.shape[0], data.shape[1]
    out = torch.empty((B, C, *outsize), device=data.device, dtype=torch.float32)
    with _on(data.device):
        _check(lib().cpab_b200_interpolate(
            ndim, _ptr(data), B, C, _i64_array(data.shape[2:]), _ptr(grid), _i64_array(outsize),
            _ptr(out), _stream(data.device)))
    return out


def interpolate_backward(ndim, data, grid, outsize, grad_out, want_grid, want_data):
    _require(data, "data")
    _require(grid, "grid")
    _require(grad_out, "grad")
    B, C = data.shape[0], data.shape[1]
    gg = torch.empty_like(grid) if want_grid else None
    gd = torch.empty_like(data) if want_data else None
    with _on(data.device):
        _check(lib().cpab_b200_interpolate_backward(
            ndim, _ptr(data), B, C, _i64_array(data.shape[2:]), _ptr(grid), _i64_array(outsize),
            _ptr(grad_out), _ptr(gg), _ptr(gd), _stream(data.device)))
    return gg, gd


def transform_data(ndim, nc, outsize, axes, trels, As, nstepsolver, adaptive, data, order=None):
    """Fused transform_data: returns (out [n_theta, C, *outsize], grid_t
    [n_theta, ndim, prod(outsize)] in processing order)."""
    _require(data, "data")
    _require(As, "As")
    _require(trels, "Trels")
    _require(axes, "mesh axes")
    n_theta, C = As.shape[0], data.shape[1]
    P = int(np_prod(outsize))
    out = torch.empty((n_theta, C, *outsize), device=As.device, dtype=torch.float32)
    grid_t = torch.empty((n_theta, ndim, P), device=As.device, dtype=torch.float32)
    with _on(As.device):
        _check(lib().cpab_b200_transform_data(
            ndim, _i32_array(nc), _i64_array(outsize), _ptr(axes), _ptr(order), _ptr(trels),
            _ptr(As), n_theta,
            int(nstepsolver), int(adaptive), _ptr(data), C, _i64_array(data.shape[2:]),
            _ptr(grid_t), _ptr(out), _stream(As.device)))
    return out, grid_t


def transform_data_backward(ndim, nc, outsize, axes, As, nstepsolver, adaptive, data, grid_t,
                            grad_out, want_data, order=None):
    """Returns (moments [n_theta, nC, ppc], grad_data or None)."""
    _require(data, "data")
    _require(As, "As")
    _require(grid_t, "grid_t")
    _require(grad_out, "grad")
    n_theta, nC, C = As.shape[0], As.shape[1], data.shape[1]
    moments = torch.empty((n_theta, nC, ndim * (ndim + 1)), device=As.device, dtype=torch.float32)
    gd = torch.empty_like(data) if want_data else None
    with _on(As.device):
        _check(lib().cpab_b200_transform_data_backward(
            ndim, _i32_array(nc), _i64_array(outsize), _ptr(axes), _ptr(order), _ptr(As), n_theta,
            int(nstepsolver), int(adaptive), _ptr(data), C, _i64_array(data.shape[2:]),
            _ptr(grid_t), _ptr(grad_out), _ptr(moments), _ptr(gd), _stream(As.device)))
    return moments, gd


def _data_batched(data, n_theta):
    """1 when data holds one image per transformation, 0 for one shared image."""
    if data.shape[0] not in (1, n_theta):
        raise ValueError("data must hold 1 or n_theta = %d images, got %d" % (n_theta, data.shape[0]))
    return int(data.shape[0] == n_theta)


def warp(ndim, nc, outsize, axes, trels, As, n_stages, nstepsolver, adaptive, data, padding,
         order=None):
    """Fused spatial-transformer warp of n_theta = As.shape[0] / n_stages
    transformations; data is [n_theta, C, *in_size] or [1, C, *in_size]
    (shared).  Returns (out [n_theta, C, *outsize], grid_t [n_theta, ndim, P],
    stage_points [n_stages-1, n_theta, ndim, P] or None)."""
    _require(data, "data")
    _require(As, "As")
    _require(trels, "Trels")
    _require(axes, "mesh axes")
    n_theta, C = As.shape[0] // n_stages, data.shape[1]
    P = int(np_prod(outsize))
    out = torch.empty((n_theta, C, *outsize), device=As.device, dtype=torch.float32)
    grid_t = torch.empty((n_theta, ndim, P), device=As.device, dtype=torch.float32)
    sp = (torch.empty((n_stages - 1, n_theta, ndim, P), device=As.device, dtype=torch.float32)
          if n_stages > 1 else None)
    batched = _data_batched(data, n_theta)
    with _on(As.device):
        _check(lib().cpab_b200_warp(
            ndim, _i32_array(nc), _i64_array(outsize), _ptr(axes), _ptr(order), _ptr(trels),
            _ptr(As), n_stages, n_theta, int(nstepsolver), int(adaptive), _ptr(data), batched, C,
            _i64_array(data.shape[2:]), int(padding), _ptr(sp), _ptr(grid_t), _ptr(out),
            _stream(As.device)))
    return out, grid_t, sp


def warp_backward(ndim, nc, outsize, axes, As, n_stages, nstepsolver, adaptive, data, padding,
                  stage_points, grid_t, grad_out, want_data, order=None):
    """Returns (moments [n_stages * n_theta, nC, ppc], grad_data shaped like
    data, or None)."""
    _require(data, "data")
    _require(As, "As")
    _require(grid_t, "grid_t")
    _require(grad_out, "grad")
    n_theta, nC, C = As.shape[0] // n_stages, As.shape[1], data.shape[1]
    moments = torch.empty((n_stages * n_theta, nC, ndim * (ndim + 1)), device=As.device,
                          dtype=torch.float32)
    gd = torch.empty_like(data) if want_data else None
    batched = _data_batched(data, n_theta)
    with _on(As.device):
        _check(lib().cpab_b200_warp_backward(
            ndim, _i32_array(nc), _i64_array(outsize), _ptr(axes), _ptr(order), _ptr(As),
            n_stages, n_theta, int(nstepsolver), int(adaptive), _ptr(data), batched, C,
            _i64_array(data.shape[2:]), int(padding), _ptr(stage_points), _ptr(grid_t),
            _ptr(grad_out), _ptr(moments), _ptr(gd), _stream(As.device)))
    return moments, gd


def forward_chain(ndim, nc, points, batched, trels, As, n_stages, nstepsolver, adaptive,
                  order=None):
    """Fused chain; trels/As [n_stages * n_theta, nC, ...] stage-major.  Returns
    (out [n_theta, ndim, nP], stage_points [n_stages-1, n_theta, ndim, nP] or None)."""
    _require(points, "points")
    _require(As, "As")
    _require(trels, "Trels")
    n_theta = As.shape[0] // n_stages
    nP = points.shape[-1]
    out = torch.empty((n_theta, ndim, nP), device=As.device, dtype=torch.float32)
    sp = (torch.empty((n_stages - 1, n_theta, ndim, nP), device=As.device, dtype=torch.float32)
          if n_stages > 1 else None)
    with _on(As.device):
        _check(lib().cpab_b200_forward_chain(
            ndim, _i32_array(nc), _ptr(points), nP, int(batched), _ptr(order), _ptr(trels),
            _ptr(As), n_stages, n_theta, int(nstepsolver), int(adaptive), _ptr(sp), _ptr(out),
            _stream(As.device)))
    return out, sp


def backward_chain(ndim, nc, points, batched, As, n_stages, grad_out, stage_points, nstepsolver,
                   adaptive, want_points, order=None):
    """Returns (moments [n_stages * n_theta, nC, ppc], grad_points or None)."""
    _require(points, "points")
    _require(As, "As")
    _require(grad_out, "grad")
    n_theta, nC = As.shape[0] // n_stages, As.shape[1]
    nP = points.shape[-1]
    moments = torch.empty((n_stages * n_theta, nC, ndim * (ndim + 1)), device=As.device,
                          dtype=torch.float32)
    gp = (torch.empty((n_theta, ndim, nP), device=As.device, dtype=torch.float32)
          if want_points else None)
    with _on(As.device):
        _check(lib().cpab_b200_backward_chain(
            ndim, _i32_array(nc), _ptr(points), nP, int(batched), _ptr(order), _ptr(As), n_stages,
            n_theta, _ptr(grad_out), _ptr(stage_points), int(nstepsolver), int(adaptive),
            _ptr(moments), _ptr(gp), _stream(As.device)))
    return moments, gp


# ---------------------------------------------------------------------------
# Operators of the sequence networks.
# ---------------------------------------------------------------------------

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _dtype(t, name):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    return code


def _like(t, x, name, dtype, shape):
    if t.device != x.device:
        raise RuntimeError("%s is on %s, x on %s" % (name, t.device, x.device))
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))


def _cuda(x):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor (no CPU path)")
    _dtype(x, "x")


def _adjacent(t):
    """t with the last axis' elements adjacent in memory."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def needs_grad(*tensors):
    """Whether the call has to go through its node, which refuses forward mode."""
    return has_tangent(*tensors) or (
        torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def has_tangent(*tensors):
    """Whether a forward-mode derivative flows into one of them."""
    return any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None
               for t in tensors)


def _written(*tensors):
    """Counts a write through a raw pointer as torch's own operations count
    theirs, so that a backward through the old value raises."""
    torch.autograd.graph.increment_version(tensors)


def check_scan(x, gate, h0, lengths):
    _cuda(x)
    if x.dim() != 3:
        raise ValueError("x must be [B, T, D], got %s" % (tuple(x.shape),))
    if gate is not None:
        _like(gate, x, "gate", x.dtype, x.shape)
    elif x.shape[2] % 2:
        raise ValueError("x without a gate must be [B, T, 2 D], got %s" % (tuple(x.shape),))
    D = x.shape[2] if gate is not None else x.shape[2] // 2
    if h0 is not None:
        _like(h0, x, "h0", torch.float32, (x.shape[0], D))
    if lengths is not None:
        _like(lengths, x, "lengths", torch.int32, (x.shape[0],))


def _scan_input(x, gate):
    """(tensors to keep alive, B, T, D, the C arguments of x and gate)."""
    xa = _adjacent(x)
    sx = (xa.stride(0), xa.stride(1))
    if gate is not None:
        ga = _adjacent(gate)
        return (xa, ga), x.shape[0], x.shape[1], x.shape[2], (
            _ptr(xa), *sx, _ptr(ga), ga.stride(0), ga.stride(1))
    D = x.shape[2] // 2
    return (xa,), x.shape[0], x.shape[1], D, (_ptr(xa), *sx, _ptr(xa) + D * x.element_size(), *sx)


def _contiguous(t):
    return t.contiguous() if t is not None else None


def _scan_workspace(x, B, T, D):
    n = lib().cpab_b200_gated_scan_workspace(_dtype(x, "x"), B, T, D)
    return torch.empty(n, device=x.device, dtype=torch.float32)


def gated_scan(x, gate, h0, lengths, keep):
    """(h, last, states or None); states only when `keep` (for the backward)."""
    alive, B, T, D, args = _scan_input(x, gate)
    f32 = dict(device=x.device, dtype=torch.float32)
    h = torch.empty((B, T, D), device=x.device, dtype=x.dtype)
    last = torch.empty((B, D), **f32)
    c = lib().cpab_b200_gated_scan_chunk()
    states = torch.empty((B, (T + c - 1) // c, D), **f32) if keep else None
    h0, lengths = _contiguous(h0), _contiguous(lengths)
    with _on(x.device):
        work = _scan_workspace(x, B, T, D)
        _check(lib().cpab_b200_gated_scan(
            _dtype(x, "x"), *args, B, T, D, _ptr(lengths), _ptr(h0), _ptr(h), _ptr(last),
            _ptr(states), _ptr(work), _stream(x.device)))
    return h, last, states


def gated_scan_backward(x, gate, lengths, states, dh, dlast, want_h0):
    """(grad_x, grad_gate or None, grad_h0 or None)."""
    alive, B, T, D, args = _scan_input(x, gate)
    dx = torch.empty((B, T, D if gate is not None else 2 * D), device=x.device, dtype=x.dtype)
    dg = torch.empty((B, T, D), device=x.device, dtype=x.dtype) if gate is not None else None
    dgp = _ptr(dg) if dg is not None else _ptr(dx) + D * x.element_size()
    dgs = dg if dg is not None else dx
    dh0 = torch.empty((B, D), device=x.device, dtype=torch.float32) if want_h0 else None
    dh, dlast, lengths = _contiguous(dh), _contiguous(dlast), _contiguous(lengths)
    with _on(x.device):
        work = _scan_workspace(x, B, T, D)
        _check(lib().cpab_b200_gated_scan_backward(
            _dtype(x, "x"), *args, B, T, D, _ptr(lengths), _ptr(states), _ptr(dh), _ptr(dlast),
            _ptr(dx), dx.stride(0), dx.stride(1), dgp, dgs.stride(0), dgs.stride(1), _ptr(dh0),
            _ptr(work), _stream(x.device)))
    return dx, dg, dh0


def gated_scan_step(x, gate, state, slots):
    _cuda(x)
    if has_tangent(x, gate, state):
        raise RuntimeError("gated_scan_step has no gradient, of forward mode neither")
    if x.dim() != 2:
        raise ValueError("x must be [B, D], got %s" % (tuple(x.shape),))
    if gate is not None:
        _like(gate, x, "gate", x.dtype, x.shape)
    elif x.shape[1] % 2:
        raise ValueError("x without a gate must be [B, 2 D], got %s" % (tuple(x.shape),))
    B, D = x.shape[0], x.shape[1] if gate is not None else x.shape[1] // 2
    if state.dim() != 2 or (slots is None and state.shape[0] != B):
        raise ValueError("state must be [rows, D] (rows = B without slots), got %s"
                         % (tuple(state.shape),))
    _like(state, x, "state", torch.float32, (state.shape[0], D))
    if not state.is_contiguous():
        raise ValueError("state must be contiguous (it is updated in place)")
    if slots is not None:
        _like(slots, x, "slots", torch.int32, (B,))
    xa = _adjacent(x)
    ga = _adjacent(gate) if gate is not None else None
    slots = _contiguous(slots)
    h = torch.empty((B, D), device=x.device, dtype=x.dtype)
    gp = _ptr(ga) if ga is not None else _ptr(xa) + D * x.element_size()
    _written(state)
    with _on(x.device):
        _check(lib().cpab_b200_gated_scan_step(
            _dtype(x, "x"), _ptr(xa), xa.stride(0), gp, (ga if ga is not None else xa).stride(0), B,
            D, _ptr(slots), state.shape[0], _ptr(state), _ptr(h), _stream(x.device)))
    return h


def check_norm(x, weight, residual):
    _cuda(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [..., D] with D > 0, got %s" % (tuple(x.shape),))
    for t, name, shape in ((weight, "weight", (x.shape[-1],)), (residual, "residual", x.shape)):
        if t is not None:
            if t.dtype not in (torch.float32, x.dtype):
                raise TypeError("%s must be float32 or of x's type, got %s" % (name, t.dtype))
            _like(t, x, name, t.dtype, shape)


def _rows(t):
    if t is None:
        return None
    return _adjacent(t if t.dim() == 2 else t.reshape(t.numel() // t.shape[-1], t.shape[-1]))


def _norm_args(x, weight, residual, eps):
    """(tensors to keep alive, the C arguments up to eps)."""
    xr, rr, w = _rows(x), _rows(residual), weight.contiguous()
    s = residual if residual is not None else x
    return (xr, rr, w), (
        _dtype(x, "x"), _dtype(s, "residual"), _dtype(w, "weight"), _ptr(xr), xr.stride(0), _ptr(rr),
        rr.stride(0) if rr is not None else 0, _ptr(w), xr.shape[0], xr.shape[1], eps)


def rms_norm(x, weight, residual, eps, keep):
    """(y, sum or None, rstd or None); rstd only when `keep` (for the backward)."""
    alive, args = _norm_args(x, weight, residual, eps)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    s = torch.empty(x.shape, device=x.device, dtype=residual.dtype) if residual is not None else None
    rstd = torch.empty(args[8], device=x.device, dtype=torch.float32) if keep else None
    with _on(x.device):
        _check(lib().cpab_b200_rms_norm(*args, _ptr(y), _ptr(s), _ptr(rstd), _stream(x.device)))
    return y, s, rstd


def rms_norm_quantized(x, weight, residual, eps):
    """(q, scale) or (q, scale, sum)."""
    if has_tangent(x, weight, residual):
        raise RuntimeError("rms_norm_quantized has no gradient, of forward mode neither")
    alive, args = _norm_args(x, weight, residual, eps)
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    s = torch.empty(x.shape, device=x.device, dtype=residual.dtype) if residual is not None else None
    with _on(x.device):
        _check(lib().cpab_b200_rms_norm_quantized(*args, _ptr(q), _ptr(scale), _ptr(s),
                                                  _stream(x.device)))
    return (q, scale) if s is None else (q, scale, s)


def rms_norm_backward(s, weight, rstd, gy, gs, x_type, want_weight):
    """(grad_x, grad_residual, grad_weight or None); the first two are one
    tensor where their types are one."""
    rows, w, gy, gs = _rows(s), weight.contiguous(), gy.contiguous(), _contiguous(gs)
    n, D = rows.shape
    dx = torch.empty(s.shape, device=s.device, dtype=x_type)
    dres = torch.empty(s.shape, device=s.device, dtype=s.dtype) if s.dtype != x_type else None
    dw = torch.empty_like(w) if want_weight else None
    dt = _dtype(dx, "x")
    work = (torch.empty(lib().cpab_b200_rms_norm_workspace(dt, n, D), device=s.device,
                        dtype=torch.float32) if want_weight else None)
    with _on(s.device):
        _check(lib().cpab_b200_rms_norm_backward(
            dt, _dtype(s, "residual"), _dtype(w, "weight"), _ptr(rows), rows.stride(0), _ptr(w),
            _ptr(rstd), n, D, _ptr(gy), _ptr(gs), _ptr(dx), _ptr(dres), _ptr(work), _ptr(dw),
            _stream(s.device)))
    return dx, (dres if dres is not None else dx), dw


def _dense(t):
    """Whether t's elements fill their span of memory, in some order of its axes."""
    span = 1
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != span:
            return t.numel() == 0
        span *= n
    return True


class _AdamWTensor(ctypes.Structure):
    """cpab_adamw_tensor."""
    _fields_ = ([(k, _p) for k in ("param", "grad", "exp_avg", "exp_avg_sq", "scales", "step",
                                   "lr_device")]
                + [("numel", _c_i64), ("dtype", ctypes.c_int32), ("state_bits", ctypes.c_int32)]
                + [(k, ctypes.c_double) for k in ("lr", "beta1", "beta2", "eps", "weight_decay")])


def adamw(params, grads, exp_avgs, exp_avg_sqs, scales, steps, counts, hyper, lrs, seed, workspace):
    """counts[g] tensors of group g one after another; hyper: each group's (lr,
    beta1, beta2, eps, weight_decay) one after another; lrs: each group's
    learning rate on the device, or None."""
    device = params[0].device
    if not params[0].is_cuda:
        raise RuntimeError("params must be CUDA tensors (no CPU path)")
    if not (len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs) == len(steps)) or \
            len(scales) not in (0, len(params)):
        raise ValueError("adamw: lists of different lengths")
    if any(lr is not None and (lr.device != device or lr.dtype != torch.float32 or lr.numel() != 1)
           for lr in lrs):
        raise RuntimeError("adamw: a learning rate on the device must be one float32 on the "
                           "parameters' device, %s" % device)
    table, alive, k = (_AdamWTensor * len(params))(), [], 0
    for group, n in enumerate(counts):
        for _ in range(n):
            p, g, m, v, step = params[k], grads[k], exp_avgs[k], exp_avg_sqs[k], steps[k]
            if any(t.device != device for t in (p, g, m, v, step)):
                raise RuntimeError("adamw: tensor %d: all tensors must be on one device" % k)
            if g.dtype != p.dtype:
                raise TypeError("adamw: tensor %d: gradient of type %s for a parameter of type %s"
                                % (k, g.dtype, p.dtype))
            if v.dtype != m.dtype or m.dtype not in (torch.float32, torch.float8_e4m3fn):
                raise TypeError("adamw: tensor %d: states must be float32, or both float8_e4m3fn" % k)
            if step.dtype != torch.float32 or step.numel() != 1:
                raise TypeError("adamw: tensor %d: step must be one float32" % k)
            if not (g.shape == p.shape == m.shape == v.shape):
                raise ValueError("adamw: tensor %d: parameter, gradient and states must have one "
                                 "shape" % k)
            alike = ((m.is_contiguous() and v.is_contiguous()) if p.is_contiguous() else
                     m.stride() == p.stride() == v.stride())
            if not _dense(p) or not alike:
                raise ValueError("adamw: tensor %d: parameter and states must be dense and laid out "
                                 "alike" % k)
            if not (g.is_contiguous() if p.is_contiguous() else g.stride() == p.stride()):
                g = torch.empty_like(p).copy_(g)
                alive.append(g)
            eight, sc = m.dtype == torch.float8_e4m3fn, None
            if eight:
                blocks = (p.numel() + 255) // 256
                sc = scales[k] if scales else None
                if sc is None or sc.device != device or sc.dtype != torch.float32 or \
                        not sc.is_contiguous() or sc.numel() != 2 * blocks:
                    raise ValueError("adamw: tensor %d: 8-bit states need float32 scales [%d, 2]"
                                     % (k, blocks))
                _written(sc)
            _written(p, m, v, step)
            t = table[k]
            t.param, t.grad, t.exp_avg, t.exp_avg_sq = _ptr(p), _ptr(g), _ptr(m), _ptr(v)
            t.scales, t.step, t.lr_device = _ptr(sc), _ptr(step), _ptr(lrs[group])
            t.numel, t.dtype, t.state_bits = p.numel(), _dtype(p, "a parameter"), 8 if eight else 32
            t.lr, t.beta1, t.beta2, t.eps, t.weight_decay = hyper[5 * group:5 * group + 5]
            k += 1
    with _on(device):
        _check(lib().cpab_b200_adamw(ctypes.byref(table), len(params), seed & 0xFFFFFFFF,
                                     _ptr(workspace), _stream(device)))


# Projections in 8 bits.

class _Quantized(ctypes.Structure):
    """cpab_quantized."""
    _fields_ = [("codes", _p), ("row", _c_i64), ("scale", _p), ("scale_row", _c_i64)]


def check_quantize(x):
    _cuda(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [..., K] with K > 0, got %s" % (tuple(x.shape),))


def check_linear(x, weight, bias):
    check_quantize(x)
    if weight.dim() != 2:
        raise ValueError("weight must be [N, K], got %s" % (tuple(weight.shape),))
    for t, name, shape in ((weight, "weight", (weight.shape[0], x.shape[-1])),
                           (bias, "bias", (weight.shape[0],))):
        if t is not None:
            if t.dtype not in (torch.float32, x.dtype):
                raise TypeError("%s must be float32 or of x's type, got %s" % (name, t.dtype))
            _like(t, x, name, t.dtype, shape)


def _codes(lead, K, device):
    """Codes [*lead, K] whose rows begin on multiples of 16 bytes, and scales
    [*lead, ceil(K / 128)] whose rows begin on multiples of 4."""
    blocks = (K + 127) // 128
    q = torch.empty((*lead, (K + 15) // 16 * 16), device=device, dtype=torch.float8_e4m3fn)[..., :K]
    s = torch.empty((*lead, (blocks + 3) // 4 * 4), device=device, dtype=torch.uint8)[..., :blocks]
    return q, s.view(torch.float8_e8m0fnu)


def _pitch(t):
    """The distance of rows of codes or scales as _codes lays them out."""
    unit = 16 if t.dtype == torch.float8_e4m3fn else 4
    return (t.shape[-1] + unit - 1) // unit * unit


def quantize_blocks(x, rows=True, transposed=False, sum_dtype=None):
    """(q, scale, qt, scale_t, sums), None where not asked for."""
    xr = _rows(x)
    R, K = xr.shape
    q = s = qt = st = sums = work = None
    if rows:
        q, s = _codes(x.shape[:-1], K, x.device)
    if transposed:
        qt, st = _codes((K,), R, x.device)
    if sum_dtype is not None:
        sums = torch.empty(K, device=x.device, dtype=sum_dtype)
        work = torch.empty(lib().cpab_b200_quantize_blocks_workspace(R, K), device=x.device,
                           dtype=torch.float32)
    with _on(x.device):
        _check(lib().cpab_b200_quantize_blocks(
            _dtype(x, "x"), _ptr(xr), xr.stride(0), R, K, _ptr(q), _pitch(q) if rows else 0, _ptr(s),
            _pitch(s) if rows else 0, _ptr(qt), _pitch(qt) if transposed else 0, _ptr(st),
            _pitch(st) if transposed else 0, _DTYPES[sum_dtype] if sums is not None else 0,
            _ptr(sums), _ptr(work), _stream(x.device)))
    return q, s, qt, st, sums


def _quantized(q, scale, name):
    """(tensors to keep alive, rows, K, cpab_quantized) of codes [..., K]."""
    if q.dtype != torch.float8_e4m3fn:
        raise TypeError("%s must be float8_e4m3fn, got %s" % (name, q.dtype))
    if q.dim() < 1 or q.shape[-1] < 1:
        raise ValueError("%s must be [..., K] with K > 0, got %s" % (name, tuple(q.shape)))
    K, lead = q.shape[-1], tuple(q.shape[:-1])
    blocks = (K + 127) // 128
    if scale.device != q.device:
        raise RuntimeError("%s's scale is on %s, the codes on %s" % (name, scale.device, q.device))
    if scale.dtype not in (torch.float8_e8m0fnu, torch.float32):
        raise TypeError("%s's scale must be float8_e8m0fnu (for each 128 codes) or float32 (for each row), "
                        "got %s" % (name, scale.dtype))
    per_row = scale.dtype == torch.float32
    want = lead if per_row else (*lead, blocks)
    if tuple(scale.shape) != want:
        raise ValueError("%s's scale must have shape %s, got %s" % (name, want, tuple(scale.shape)))
    qr = q if q.dim() == 2 else q.reshape(-1, K)
    rows = qr.shape[0]
    if K > 1 and qr.stride(1) != 1:
        qr = _codes((rows,), K, q.device)[0].copy_(qr)
    if (rows > 1 and (qr.stride(0) % 16 or qr.stride(0) < K)) or qr.data_ptr() % 16:
        src, qr = qr, _codes((rows,), K, q.device)[0]
        with _on(q.device):
            _check(lib().cpab_b200_lay_out_codes(
                1, (_p * 1)(_ptr(src)), (_c_i64 * 1)(src.stride(0)), (_c_i64 * 1)(rows), (_p * 1)(_ptr(qr)), K,
                _stream(q.device)))
    if per_row:
        sr = scale.reshape(-1).contiguous()
        scale_row = 0
    else:
        sr = scale if scale.dim() == 2 else scale.reshape(-1, blocks)
        if (blocks > 1 and sr.stride(1) != 1) or (rows > 1 and sr.stride(0) < blocks):
            sr = sr.contiguous()
        scale_row = sr.stride(0) if rows > 1 else (blocks + 3) // 4 * 4
    row = qr.stride(0) if rows > 1 else (K + 15) // 16 * 16
    return (qr, sr), rows, K, _Quantized(_ptr(qr), row, _ptr(sr), scale_row)


def matmul_quantized(q, scale, weight, weight_scale, bias, dtype):
    if not q.is_cuda:
        raise RuntimeError("q must be a CUDA tensor (no CPU path)")
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float32, float16 or bfloat16, got %s" % dtype)
    if weight.dim() != 2:
        raise ValueError("weight must be [N, K], got %s" % (tuple(weight.shape),))
    if weight.device != q.device:
        raise RuntimeError("weight is on %s, q on %s" % (weight.device, q.device))
    if has_tangent(scale, weight_scale, bias):
        raise RuntimeError("matmul_quantized has no gradient, of forward mode neither")
    alive, M, K, x = _quantized(q, scale, "q")
    alive_w, N, Kw, w = _quantized(weight, weight_scale, "weight")
    if Kw != K:
        raise ValueError("weight must be [N, %d], got %s" % (K, tuple(weight.shape)))
    if bias is not None:
        if bias.dtype not in (torch.float32, dtype):
            raise TypeError("bias must be float32 or of the result's type, got %s" % bias.dtype)
        _like(bias, q, "bias", bias.dtype, (N,))
        bias = bias.contiguous()
    y = torch.empty((*q.shape[:-1], N), device=q.device, dtype=dtype)
    with _on(q.device):
        floats = lib().cpab_b200_matmul_quantized_workspace(M, N, K)
        work = torch.empty(floats, device=q.device, dtype=torch.float32) if floats else None
        _check(lib().cpab_b200_matmul_quantized(
            _DTYPES[dtype], ctypes.byref(x), ctypes.byref(w), M, N, K,
            _DTYPES[bias.dtype] if bias is not None else _DTYPES[dtype], _ptr(bias), _ptr(y), N,
            _ptr(work), _stream(q.device)))
    return y


# Orthogonalised directions.

class _MuonTensor(ctypes.Structure):
    """cpab_muon_tensor."""
    _fields_ = [("param", _p), ("grad", _p), ("momentum", _p), ("rows", _c_i64), ("columns", _c_i64),
                ("dtype", ctypes.c_int32)]


def _doubles(values):
    return (ctypes.c_double * 3)(*values)


def orthogonalize(x, steps, coefficients, eps):
    _cuda(x)
    if has_tangent(x):
        raise RuntimeError("orthogonalize has no gradient, of forward mode neither")
    if x.dim() < 2:
        raise ValueError("x must be [..., m, n], got %s" % (tuple(x.shape),))
    xc = x.contiguous()
    m, n = x.shape[-2:]
    batch = x.numel() // (m * n) if x.numel() else 0
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    dt = _dtype(x, "x")
    with _on(x.device):
        work = torch.empty(lib().cpab_b200_orthogonalize_workspace(dt, batch, m, n), device=x.device,
                           dtype=torch.uint8)
        _check(lib().cpab_b200_orthogonalize(dt, _ptr(xc), batch, m, n, steps, _doubles(coefficients), eps,
                                             _ptr(out), _ptr(work), _stream(x.device)))
    return out


def muon(params, grads, momenta, lr, lr_device, momentum, nesterov, weight_decay, steps, coefficients,
         eps, adjust):
    """lr_device: the learning rate as one float32 on the device, or None."""
    if not (len(params) == len(grads) == len(momenta)):
        raise ValueError("muon: lists of different lengths")
    if not params:
        return
    device = params[0].device
    if not params[0].is_cuda:
        raise RuntimeError("params must be CUDA tensors (no CPU path)")
    if lr_device is not None and (lr_device.device != device or lr_device.dtype != torch.float32
                                  or lr_device.numel() != 1):
        raise RuntimeError("muon: a learning rate on the device must be one float32 on the parameters' "
                           "device, %s" % device)
    table, alive = (_MuonTensor * len(params))(), []
    for k, (p, g, m) in enumerate(zip(params, grads, momenta)):
        if any(t.device != device for t in (p, g, m)):
            raise RuntimeError("muon: tensor %d: all tensors must be on one device" % k)
        if g.dtype != p.dtype:
            raise TypeError("muon: tensor %d: gradient of type %s for a parameter of type %s"
                            % (k, g.dtype, p.dtype))
        if m.dtype != torch.float32:
            raise TypeError("muon: tensor %d: momentum must be float32, got %s" % (k, m.dtype))
        if p.dim() != 2 or not (g.shape == p.shape == m.shape):
            raise ValueError("muon: tensor %d: parameter, gradient and momentum must be matrices of one "
                             "shape, got %s" % (k, tuple(p.shape)))
        if not p.is_contiguous() or not m.is_contiguous():
            raise ValueError("muon: tensor %d: parameter and momentum must be contiguous" % k)
        if not g.is_contiguous():
            g = g.contiguous()
            alive.append(g)
        table[k] = _MuonTensor(_ptr(p), _ptr(g), _ptr(m), p.shape[0], p.shape[1], _dtype(p, "a parameter"))
        _written(p, m)
    with _on(device):
        work = torch.empty(lib().cpab_b200_muon_workspace(ctypes.byref(table), len(params)), device=device,
                           dtype=torch.uint8)
        _check(lib().cpab_b200_muon(ctypes.byref(table), len(params), lr, _ptr(lr_device), momentum,
                                    int(nesterov), weight_decay, steps, _doubles(coefficients), eps, adjust,
                                    _ptr(work), _stream(device)))
