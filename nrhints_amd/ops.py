"""Thin tensor-level wrappers over the fine-grained C entry points (include/nrhints_hip.h).

``NeuSHintRenderer.forward`` does not use these (it makes one fused C call per chunk); they exist so that each
kernel can be parity-tested in isolation and so that callers such as mesh extraction can query the SDF alone.
All tensors are float32, contiguous, on the GPU.  No fallback: errors raise.

The last section holds the layer operators, which take networks and tables of ANY shape in float32, float16 or bfloat16: ``linear`` (a
layer's product with bias, activation and residual) and ``embedding`` (rows of a table, scaled) with their gradients.  They work on
plain tensors and record no autograd graph; ``nrhints_amd.layers`` wraps them for autograd.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, packing


def _scratch(device) -> torch.Tensor:
    lib = _lib.load()
    n = lib.nrh_mlp_grid() * _lib.param_sizes()[7] * packing.SDF_SCRATCH_FLOATS_PER_WAVE
    return torch.empty(n, dtype=torch.float32, device=device)


def _wptr(w):
    """Packed weights: float32 (precision 0) or float16 pairs (precision 1, f16x3)."""
    return _lib.ptr(w, w.dtype), (0 if w.dtype == torch.float32 else 1)


@_lib.on_tensor_device
def sdf_eval(mode: int, sdf_w, sdf_b, sdf_head, ro, rd, t, n_per_ray: int, t_stride: Optional[int] = None,
             scratch: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """SDF (mode 0), + gradient (mode 1), + feature (mode 2) at points ro[ray] + rd[ray] * t[ray, j].

    Returns (sdf [nrays, n_per_ray], grad [nrays*n_per_ray, 3] | None, feat tiles | None)."""
    lib = _lib.load()
    nrays = ro.shape[0]
    t_stride = n_per_ray if t_stride is None else t_stride
    dev = ro.device
    sdf = torch.empty(nrays, n_per_ray, dtype=torch.float32, device=dev)
    npts = nrays * n_per_ray
    grad = torch.empty(npts, 3, dtype=torch.float32, device=dev) if mode >= 1 else None
    feat = torch.empty(((npts + 15) // 16) * 4096, dtype=torch.float32, device=dev) if mode == 2 else None
    if mode >= 1 and scratch is None:
        scratch = _scratch(dev)
    P = _lib.ptr
    wp, prec = _wptr(sdf_w)
    rc = lib.nrh_sdf_eval(prec, mode, wp, P(sdf_b), P(sdf_head), P(ro), P(rd), P(t), t_stride, n_per_ray, nrays,
                          P(sdf), n_per_ray, P(grad), P(feat), P(scratch) if mode >= 1 else None, _lib.stream_handle())
    _lib.check(rc, "nrh_sdf_eval")
    return sdf, grad, feat


@_lib.on_tensor_device
def sdf_eval_wide(mode: int, sdf_w32, sdf_tab32, ro, rd, t, n_per_ray: int, t_stride: Optional[int] = None,
                  scratch: Optional[torch.Tensor] = None, one_term: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``sdf_eval`` through the wide f16x3 kernels (csrc/nrh_sdf32.hip); sdf_w32 / sdf_tab32 from packing32.pack_sdf32.
    mode 3 (wide only): sdf + the derivative along the ray in forward mode; ``grad`` = rd * (d sdf / dt) / |rd|^2.
    ``one_term``: their single-pass builds (precision "f16": one fp16 MFMA per K step, csrc/nrh_wide1.hip), same buffers."""
    lib = _lib.load()
    nrays = ro.shape[0]
    t_stride = n_per_ray if t_stride is None else t_stride
    dev = ro.device
    sdf = torch.empty(nrays, n_per_ray, dtype=torch.float32, device=dev)
    npts = nrays * n_per_ray
    grad = torch.empty(npts, 3, dtype=torch.float32, device=dev) if mode >= 1 else None
    feat = torch.empty(((npts + 15) // 16) * 4096, dtype=torch.float32, device=dev) if mode == 2 else None
    if mode in (1, 2) and scratch is None:
        scratch = _scratch(dev)
    if sdf_w32.numel() * sdf_w32.element_size() != lib.nrh_sdf_wide_stream_bytes():
        raise ValueError("sdf_w32 has the wrong size for this library build")
    P = _lib.ptr
    with torch.cuda.device(dev):
        fn = lib.nrh_sdf_eval_wide_f16 if one_term else lib.nrh_sdf_eval_wide
        rc = fn(mode, P(sdf_w32, sdf_w32.dtype), P(sdf_tab32), P(ro), P(rd), P(t), t_stride, n_per_ray, nrays,
                P(sdf), n_per_ray, P(grad), P(feat), P(scratch) if mode in (1, 2) else None, _lib.stream_handle(dev))
    _lib.check(rc, "nrh_sdf_eval_wide")
    return sdf, grad, feat


@_lib.on_tensor_device
def sdf_eval_split(sdf_w, sdf_b, sdf_head, ro, rd, t, n_per_ray: int, t_stride: Optional[int] = None, tiles: int = 0) -> torch.Tensor:
    """SDF values of a small point set on the channel-split kernel (csrc/nrh_sdf_split.hip): ``sdf_eval`` mode 0 with the
    precision-1 (f16x3) packed parameters, bit-identical values, a quarter of the per-pass latency.  tiles: 0 (auto), 1 or 2."""
    lib = _lib.load()
    nrays = ro.shape[0]
    t_stride = n_per_ray if t_stride is None else t_stride
    sdf = torch.empty(nrays, n_per_ray, dtype=torch.float32, device=ro.device)
    P = _lib.ptr
    with torch.cuda.device(ro.device):
        rc = lib.nrh_sdf_eval_split(P(sdf_w, sdf_w.dtype), P(sdf_b), P(sdf_head), P(ro), P(rd), P(t), t_stride, n_per_ray, nrays,
                                    P(sdf), n_per_ray, tiles, _lib.stream_handle(ro.device))
    _lib.check(rc, "nrh_sdf_eval_split")
    return sdf


@_lib.on_tensor_device
def sdf_grad_split(sdf_w, sdf_b, sdf_head, ro, rd, t, n_per_ray: int, t_stride: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """sdf and d sdf / dx of a small point set on the channel-split kernel: ``sdf_eval`` mode 1 with the precision-1 (f16x3) packed
    parameters, bit-identical values, no scratch.  -> (sdf [nrays, n_per_ray], grad [nrays * n_per_ray, 3])."""
    lib = _lib.load()
    nrays = ro.shape[0]
    t_stride = n_per_ray if t_stride is None else t_stride
    sdf = torch.empty(nrays, n_per_ray, dtype=torch.float32, device=ro.device)
    grad = torch.empty(nrays * n_per_ray, 3, dtype=torch.float32, device=ro.device)
    P = _lib.ptr
    with torch.cuda.device(ro.device):
        rc = lib.nrh_sdf_grad_split(P(sdf_w, sdf_w.dtype), P(sdf_b), P(sdf_head), P(ro), P(rd), P(t), t_stride, n_per_ray, nrays,
                                    P(sdf), n_per_ray, P(grad), _lib.stream_handle(ro.device))
    _lib.check(rc, "nrh_sdf_grad_split")
    return sdf, grad


@_lib.on_tensor_device
def sdf_at_points(mode: int, sdf_w, sdf_b, sdf_head, pts):
    """Convenience: free points [P,3] (one 'ray' per point, t = 0)."""
    zeros = torch.zeros_like(pts)
    t = torch.zeros(pts.shape[0], dtype=torch.float32, device=pts.device)
    return sdf_eval(mode, sdf_w, sdf_b, sdf_head, pts.contiguous(), zeros, t, 1)


@_lib.on_tensor_device
def sdf_train_forward(sdf_w, sdf_b, sdf_head, pts, half_handoffs: bool = False):
    """Training forward at free points [P,3] (P % 16 == 0): -> (sdf [P,1], feat [P,256] row-major, grad [P,3], saves)
    where ``saves`` holds what ``sdf_train_backward`` and the weight-gradient GEMMs need (include/nrhints_hip.h).
    ``half_handoffs`` (f16x3, nrh_train_half_supported): saves also has ``h16`` (layers 0..6; saves["h"] then only holds layer 7) and
    ``t16`` (layers 1..7), float16 [8,P,256] in the half-tiled layout (nrh_sdf_train_forward_half)."""
    lib = _lib.load()
    n = pts.shape[0]
    dev = pts.device
    f32 = dict(dtype=torch.float32, device=dev)
    zeros3 = torch.zeros(n, 3, **f32)
    zeros1 = torch.zeros(n, **f32)
    sdf = torch.empty(n, 1, **f32)
    grad = torch.empty(n, 3, **f32)
    feat = torch.empty(n, 256, **f32)
    saves = dict(h=torch.empty(8, n, 256, **f32), s1=torch.empty(8, n, 256, **f32), t=torch.empty(8, n, 256, **f32),
                 ge=torch.empty(n, 128, **f32), zeros3=zeros3, zeros1=zeros1)
    P = _lib.ptr
    wp, prec = _wptr(sdf_w)
    if half_handoffs:
        saves["h16"] = torch.empty(8, n, 256, dtype=torch.float16, device=dev)
        saves["t16"] = torch.empty(8, n, 256, dtype=torch.float16, device=dev)
        rc = lib.nrh_sdf_train_forward_half(prec, wp, P(sdf_b), P(sdf_head), P(pts), P(zeros3), P(zeros1), 1, 1, n, P(sdf), P(grad),
                                            P(feat), P(saves["h"]), P(saves["s1"]), P(saves["t"]), P(saves["ge"]),
                                            P(saves["h16"], torch.float16), P(saves["t16"], torch.float16), _lib.stream_handle())
        _lib.check(rc, "nrh_sdf_train_forward_half")
        return sdf, feat, grad, saves
    rc = lib.nrh_sdf_train_forward(prec, wp, P(sdf_b), P(sdf_head), P(pts), P(zeros3), P(zeros1), 1, 1, n, P(sdf), P(grad),
                                   P(feat), P(saves["h"]), P(saves["s1"]), P(saves["t"]), P(saves["ge"]), _lib.stream_handle())
    _lib.check(rc, "nrh_sdf_train_forward")
    return sdf, feat, grad, saves


@_lib.on_tensor_device
def sdf_train_backward(sdf_w, wt_feat, sdf_head, ro, rd, t, n_per_ray, saves, sbar, fbar, gbar, adj_scale: float = 1.0,
                       half_handoffs: bool = False, dyn: Optional[torch.Tensor] = None):
    """The two backward sweeps at the points ro[ray] + rd[ray] * t[ray, j]
    -> dict(abar, coup, zbar [8,P,256], gebar [P,64], pbar [P,3]).  ``adj_scale``: see _lib.adjoint_scale (a training step passes
    it; 1 = the adjoints as they come, for callers whose adjoints are O(1)).
    ``half_handoffs`` (f16x3, batches with nrh_train_half_supported): layers 0..6 of abar and 1..7 of zbar leave as float16 arrays
    ``abar16`` / ``zbar16`` (half-tiled, times the step's adjoint scale, which the library takes from the seeds' range and writes to
    ``dyn`` = float32 [4], zero before its first use) INSTEAD of the float32 arrays; adj_scale is not used."""
    lib = _lib.load()
    nrays = ro.shape[0]
    n = nrays * n_per_ray
    f32 = dict(dtype=torch.float32, device=ro.device)
    out = dict(abar=torch.empty(8, n, 256, **f32), coup=torch.empty(8, n, 256, **f32), zbar=torch.empty(8, n, 256, **f32),
               gebar=torch.empty(n, 64, **f32), pbar=torch.empty(n, 3, **f32))
    P = _lib.ptr
    wp, prec = _wptr(sdf_w)
    wtp, prec2 = _wptr(wt_feat)
    if prec != prec2:
        raise ValueError("sdf_w and wt_feat are packed for different precisions")
    if half_handoffs:
        out["abar16"] = torch.empty(8, n, 256, dtype=torch.float16, device=ro.device)
        out["zbar16"] = torch.empty(8, n, 256, dtype=torch.float16, device=ro.device)
        out["dyn"] = dyn if dyn is not None else torch.zeros(4, **f32)
        rc = lib.nrh_sdf_train_backward_half(prec, wp, wtp, P(sdf_head), P(ro), P(rd), P(t), n_per_ray, n_per_ray, nrays,
                                             P(saves["s1"]), P(saves["t"]), P(gbar), P(fbar), P(sbar), P(out["abar"]), P(out["coup"]),
                                             P(out["gebar"]), P(out["zbar"]), P(out["pbar"]), P(out["abar16"], torch.float16),
                                             P(out["zbar16"], torch.float16), P(out["dyn"]), P(saves.get("t16"), torch.float16),
                                             _lib.stream_handle())
        _lib.check(rc, "nrh_sdf_train_backward_half")
        return out
    rc = lib.nrh_sdf_train_backward(prec, wp, wtp, P(sdf_head), P(ro), P(rd), P(t), n_per_ray, n_per_ray, nrays,
                                    P(saves["s1"]), P(saves["t"]), P(gbar), P(fbar), P(sbar), P(out["abar"]), P(out["coup"]),
                                    P(out["gebar"]), P(out["zbar"]), P(out["pbar"]), float(adj_scale), _lib.stream_handle())
    _lib.check(rc, "nrh_sdf_train_backward")
    return out


@_lib.on_tensor_device
def sampler_step(ro, rd, z, s, n: int, *, znew_in=None, snew_in=None, upsample_inv_s: Optional[float] = None,
                 lin16=None, finalize: bool = False, last_dist: float = 2.0 / 64, last_dist_ray=None):
    """One launch of the hierarchical sampler.  ``z``/``s`` ([nrays,128]) are updated in place by a merge.
    Returns (znew_out [nrays,16] | None, tmid | None, dists | None)."""
    lib = _lib.load()
    nrays = ro.shape[0]
    dev = ro.device
    do_merge = znew_in is not None
    merge_sdf = snew_in is not None
    do_up = upsample_inv_s is not None
    znew_out = torch.empty(nrays, 16, dtype=torch.float32, device=dev) if do_up else None
    tmid = torch.empty(nrays, 128, dtype=torch.float32, device=dev) if finalize else None
    dists = torch.empty(nrays, 128, dtype=torch.float32, device=dev) if finalize else None
    P = _lib.ptr
    rc = lib.nrh_sampler_step(P(ro), P(rd), P(z), P(s), P(znew_in), P(snew_in), P(znew_out), P(lin16),
                              P(last_dist_ray), P(tmid), P(dists), float(upsample_inv_s or 0.0), float(last_dist),
                              nrays, n, int(do_merge), int(merge_sdf), int(do_up), int(finalize), _lib.stream_handle())
    _lib.check(rc, "nrh_sampler_step")
    return znew_out, tmid, dists


@_lib.on_tensor_device
def color_eval(col_w, col_b, feat_tiles, ro, rd, tmid, nhat, raymisc, hints: bool = True) -> torch.Tensor:
    """Reflectance MLP for nrays x 128 samples -> [nrays*128, 3] (``hints=False``: the 316-input pl-naive net)."""
    lib = _lib.load()
    nrays = ro.shape[0]
    color = torch.empty(nrays * 128, 3, dtype=torch.float32, device=ro.device)
    P = _lib.ptr
    wp, prec = _wptr(col_w)
    rc = lib.nrh_color_eval(prec, int(hints), wp, P(col_b), P(feat_tiles), P(ro), P(rd), P(tmid), P(nhat), P(raymisc), nrays,
                            P(color), _lib.stream_handle())
    _lib.check(rc, "nrh_color_eval")
    return color


@_lib.on_tensor_device
def color_eval_wide(col_w32, col_tab32, part_tiles, ro, rd, tmid, nhat, raymisc) -> torch.Tensor:
    """Reflectance MLP on the wide kernel for nrays x 128 samples -> [nrays*128, 3]; ``part_tiles``: W0feat * feature as
    16-point D-layout tiles (packing.rows_to_feat_tiles); ``raymisc`` [nrays, 100]."""
    lib = _lib.load()
    nrays = ro.shape[0]
    color = torch.empty(nrays * 128, 3, dtype=torch.float32, device=ro.device)
    P = _lib.ptr
    rc = lib.nrh_color_eval_wide(P(col_w32, col_w32.dtype), P(col_tab32), P(part_tiles), P(ro), P(rd), P(tmid), P(nhat), P(raymisc),
                                 nrays, P(color), _lib.stream_handle())
    _lib.check(rc, "nrh_color_eval_wide")
    return color


@_lib.on_tensor_device
def alpha_composite(ro, rd, pl, sdf, grad, dists, mid_z, inv_s: float, cos_anneal: float = 1.0, depth_type: int = 0,
                    zero_hints: bool = False, t_rand_shadow=None):
    """The evaluation render's alpha / compositing / hit point / specular-cue stage on its own (nrh_alpha_composite =
    core_alpha_kernel) -> dict(weights, inside [n,128], nhat [n*128,3], depth, wsum [n], cue [n,4], hit, hit_normal [n,3],
    shadow_dirs [n,3], shadow_last_dist [n], shadow_z [n,128])."""
    lib = _lib.load()
    n = ro.shape[0]
    new = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=ro.device)
    lin64 = torch.linspace(0.0, 1.0, 64).to(ro.device)
    out = dict(weights=new(n, 128), inside=new(n, 128), nhat=new(n * 128, 3), depth=new(n), wsum=new(n), cue=new(n, 4),
               hit=new(n, 3), hit_normal=new(n, 3), shadow_dirs=new(n, 3), shadow_last_dist=new(n), shadow_z=torch.zeros(n, 128, dtype=torch.float32, device=ro.device))
    P = _lib.ptr
    rc = lib.nrh_alpha_composite(P(ro), P(rd), P(pl), P(sdf), P(grad), P(dists), P(mid_z), float(inv_s), float(cos_anneal), int(depth_type),
                                 int(bool(zero_hints)), P(lin64), P(t_rand_shadow), n, P(out["weights"]), P(out["inside"]), P(out["nhat"]),
                                 P(out["depth"]), P(out["wsum"]), P(out["cue"]), P(out["hit"]), P(out["hit_normal"]), P(out["shadow_dirs"]),
                                 P(out["shadow_last_dist"]), P(out["shadow_z"]), _lib.stream_handle())
    _lib.check(rc, "nrh_alpha_composite")
    return out


@_lib.on_tensor_device
def visibility(rd, pl, shadow_dirs, sdf, grad, dists, cue, inv_s: float, cos_anneal: float = 1.0, zero_hints: bool = False):
    """Shadow-ray transmittance + the reflectance net's per-ray encodings (nrh_visibility = shadow_finish_kernel)
    -> (visibilities [n], raymisc [n, RAYMISC_STRIDE])."""
    from . import packing
    lib = _lib.load()
    n = rd.shape[0]
    vis = torch.empty(n, dtype=torch.float32, device=rd.device)
    raymisc = torch.zeros(n, packing.RAYMISC_STRIDE, dtype=torch.float32, device=rd.device)
    P = _lib.ptr
    rc = lib.nrh_visibility(P(rd), P(pl), P(shadow_dirs), P(sdf), P(grad), P(dists), P(cue), float(inv_s), float(cos_anneal),
                            int(bool(zero_hints)), n, P(vis), P(raymisc), _lib.stream_handle())
    _lib.check(rc, "nrh_visibility")
    return vis, raymisc


@_lib.on_tensor_device
def color_composite(color, weights, wsum, background=None, inside=None, grad=None, nhat=None, maps: bool = False):
    """rgb = sum c w + bg (1 - sum w) (+ the two weighted normal maps) (nrh_color_composite = composite_kernel)
    -> (rgb [n,3], normal_map | None, normalized_normal_map | None)."""
    lib = _lib.load()
    n = weights.shape[0]
    new = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=weights.device)
    rgb = new(n, 3)
    nm, nnm = (new(n, 3), new(n, 3)) if maps else (None, None)
    P = _lib.ptr
    rc = lib.nrh_color_composite(P(color), P(weights), P(wsum), P(background), P(inside), P(grad), P(nhat), n, P(rgb), P(nm), P(nnm),
                                 _lib.stream_handle())
    _lib.check(rc, "nrh_color_composite")
    return rgb, nm, nnm


# ---- layer operators -------------------------------------------------------------------------------------------------------------
#: activation names of ``linear`` in the order of the C entry's codes
ACTIVATIONS = ("none", "relu", "softplus", "sigmoid", "silu", "gelu")
_ACT = {name: code for code, name in enumerate(ACTIVATIONS)}
_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _matrix(t: torch.Tensor, rows: int, cols: int, like: torch.Tensor, what: str, dtype=None):
    """``t`` as a [rows, cols] matrix of contiguous rows on ``like``'s device and of its type (or ``dtype``): -> (tensor, row stride), a
    view where the strides allow it (a column block of a wider buffer), else a copy."""
    if not isinstance(t, torch.Tensor) or t.dtype != (dtype or like.dtype) or t.device != like.device:
        raise ValueError(f"{what}: expected a {dtype or like.dtype} tensor on {like.device}, got {getattr(t, 'dtype', type(t))} on {getattr(t, 'device', None)}")
    if t.is_neg():                                         # (an imaginary part of a conjugate: the sign is a flag of the view)
        t = t.resolve_neg()
    if t.is_contiguous():
        return t, cols
    if t.dim() != 2:
        t = t.reshape(rows, cols)
    if (t.stride(1) != 1 and cols > 1) or (t.stride(0) < cols and rows > 1):
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else cols)


def _layer_input(x: torch.Tensor, what: str) -> int:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what}: expected a tensor on the GPU (there is no CPU path)")
    code = _DTYPE.get(x.dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16, got {x.dtype}")
    return code


def _linear_shapes(x, weight, activation):
    code = _ACT.get(activation)
    if code is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    dtype = _layer_input(x, "x")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear: x [..., k] and weight [n, k] with n, k >= 1, got {tuple(x.shape)} and {tuple(getattr(weight, 'shape', ()))}")
    n, k = weight.shape
    return dtype, code, x.numel() // k, n, k


class _Here:
    """``with _Here(device)``: the tensors' device current (the C entries launch on the current device) - nothing to do for the usual
    case of one device - and its current stream as an integer."""
    __slots__ = ("guard", "stream")

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
        self.stream = torch._C._cuda_getCurrentRawStream(device.index)      # current_stream(device).cuda_stream without the object

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


_WORKSPACE_BYTES = {}


def _workspace(like: torch.Tensor, entry: str, *sizes: int):
    """(workspace tensor | None, its bytes) of a C entry for these sizes; the size query is remembered, the memory is not."""
    key = (entry,) + sizes
    nbytes = _WORKSPACE_BYTES.get(key)
    if nbytes is None:
        if len(_WORKSPACE_BYTES) >= 4096:
            _WORKSPACE_BYTES.clear()
        nbytes = _WORKSPACE_BYTES[key] = getattr(_lib.load(), entry)(*sizes)
    return (like.new_empty(nbytes, dtype=torch.uint8) if nbytes > 0 else None), nbytes


def _vp(t):
    return None if t is None else t.data_ptr()


def _linear_forward(x, weight, bias, residual, activation, beta, want_dact):
    dtype, code, m, n, k = _linear_shapes(x, weight, activation)
    if code == 2 and not 0.0 < float(beta) < 1e30:
        raise ValueError("linear: softplus needs a positive beta")
    (x2, ldx), (w2, ldw) = _matrix(x, m, k, x, "x"), _matrix(weight, n, k, x, "weight")
    shape = x.shape[:-1] + (n,)
    b1, r2, ldr = None, None, 0
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"linear: bias must be [{n}], got {tuple(bias.shape)}")
        b1, _ = _matrix(bias, 1, n, x, "bias")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"linear: residual must have the output's shape {tuple(shape)}, got {tuple(residual.shape)} (it is not broadcast)")
        r2, ldr = _matrix(residual, m, n, x, "residual")
    y = x.new_empty(shape)
    dact = None
    # ReLU without a residual: y is positive exactly where the argument is (bfloat16: down to 2^-134 of it) and serves as the mask - not in
    # float16, where arguments up to 2^-25 round to zero
    masks_itself = code == 1 and residual is None and x.dtype != torch.float16
    if want_dact and code != 0 and not masks_itself:
        dact = x.new_empty(shape, dtype=x.dtype if code == 1 else torch.float32)
    ws, nbytes = _workspace(x, "nrh_linear_workspace_bytes", 0, dtype, code, m, n, k)
    with _Here(x.device) as stream:
        rc = _lib.load().nrh_linear_forward(dtype, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _vp(b1), _vp(r2), ldr, code, beta, m, n, k,
                                            y.data_ptr(), n, _vp(dact), _vp(ws), nbytes, stream)
    _lib.check(rc, "nrh_linear_forward")
    return y, (y if want_dact and masks_itself else dact)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           activation: str = "none", beta: float = 100.0) -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` in one launch (two where few rows meet a long reduction): x [..., k], weight [n, k],
    bias [n], residual of the output's shape; activation one of ``ACTIVATIONS``, softplus with ``beta`` (the SDF network's 100,
    fields/sdf_field.py:104).  One type for all tensors, float32 inside, one rounding.  Row strides are taken as they are; other
    strides are copied.  -> y [..., n] (contiguous)."""
    return _linear_forward(x, weight, bias, residual, activation, beta, False)[0]


def linear_train_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         residual: Optional[torch.Tensor] = None, activation: str = "none",
                         beta: float = 100.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``linear`` that also keeps what its gradient needs: -> (y, dact), dact = act'(x weight^T + bias) in float32, None for
    "none", a mask of x's type for "relu": y itself where there is no residual and the type is not float16 (do not change y in place before the
    backward then)."""
    return _linear_forward(x, weight, bias, residual, activation, beta, True)


def linear_backward(y_bar: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, dact: Optional[torch.Tensor], activation: str = "none",
                    want_x: bool = True, want_weight: bool = True, want_bias: bool = True):
    """Gradients of ``linear_train_forward``: -> (x_bar, weight_bar, bias_bar), None where not wanted, in the tensors' type; the
    residual's gradient is y_bar.  No floating point atomics: the same bits on every run."""
    dtype, code, m, n, k = _linear_shapes(x, weight, activation)
    shape = x.shape[:-1] + (n,)
    if y_bar.shape != shape or (dact is not None and dact.shape != shape):
        raise ValueError(f"linear_backward: y_bar and dact must be {tuple(shape)}")
    if (dact is None) != (code == 0):
        raise ValueError("linear_backward: dact (from linear_train_forward) is needed exactly when there is an activation")
    (x2, ldx), (w2, ldw), (g2, ldg) = _matrix(x, m, k, x, "x"), _matrix(weight, n, k, x, "weight"), _matrix(y_bar, m, n, x, "y_bar")
    d2, ldd = (None, 0) if dact is None else _matrix(dact, m, n, x, "dact", x.dtype if code == 1 else torch.float32)
    lib = _lib.load()
    x_bar = x.new_empty(x.shape) if want_x else None
    # (a bias alone: the column sums of ybar act' beside the weight gradient of one column of x)
    kw = k if want_weight else 1
    w_bar = x.new_empty((n, kw)) if (want_weight or want_bias) else None
    b_bar = x.new_empty((n,)) if want_bias else None
    with _Here(x.device) as stream:
        if want_x:
            ws, nbytes = _workspace(x, "nrh_linear_workspace_bytes", 1, dtype, code, m, n, k)
            _lib.check(lib.nrh_linear_backward_data(dtype, g2.data_ptr(), ldg, _vp(d2), ldd, code, w2.data_ptr(), ldw, m, n, k,
                                                    x_bar.data_ptr(), k, _vp(ws), nbytes, stream), "nrh_linear_backward_data")
        if w_bar is not None:
            ws, nbytes = _workspace(x, "nrh_linear_workspace_bytes", 2, dtype, code, m, n, kw)
            _lib.check(lib.nrh_linear_backward_weight(dtype, g2.data_ptr(), ldg, _vp(d2), ldd, code, x2.data_ptr(), ldx, m, n, kw,
                                                      w_bar.data_ptr(), kw, _vp(b_bar), _vp(ws), nbytes, stream), "nrh_linear_backward_weight")
    return x_bar, (w_bar if want_weight else None), b_bar


def _index(index, like, what):
    if not isinstance(index, torch.Tensor) or index.dtype not in (torch.int32, torch.int64) or index.device != like.device:
        raise ValueError(f"{what}: the index must be an int32 or int64 tensor on {like.device}")
    return index.resolve_neg().contiguous(), 64 if index.dtype == torch.int64 else 32


def embedding(table: torch.Tensor, index: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[index]``: table [v, d], index int32 / int64 of any shape -> [..., d] in the table's type (product in float32,
    one rounding).  An index outside [0, v) - a padded slot - gives a row of zeros and no gradient; there is no host check."""
    dtype = _layer_input(table, "table")
    if table.dim() != 2 or 0 in table.shape:
        raise ValueError(f"embedding: table must be [v, d] with v, d >= 1, got {tuple(table.shape)}")
    v, d = table.shape
    idx, bits = _index(index, table, "embedding")
    t2, ldt = _matrix(table, v, d, table, "table")
    rows = table.new_empty(index.shape + (d,))
    with _Here(table.device) as stream:
        rc = _lib.load().nrh_embedding_forward(dtype, t2.data_ptr(), ldt, v, d, idx.data_ptr(), bits, idx.numel(), scale, rows.data_ptr(), d, stream)
    _lib.check(rc, "nrh_embedding_forward")
    return rows


def embedding_backward(rows_bar: torch.Tensor, index: torch.Tensor, num_rows: int, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``embedding`` with respect to its table: [num_rows, d], row r = scale * the sum of rows_bar over the tokens with
    index r (float32 sums over tokens in their order, one rounding; zeros where there is none).  Tokens are sorted by index, nothing is
    added atomically: the same bits on every run."""
    dtype = _layer_input(rows_bar, "rows_bar")
    if rows_bar.dim() < 1 or rows_bar.shape[:-1] != index.shape or rows_bar.shape[-1] < 1 or num_rows < 1:
        raise ValueError(f"embedding_backward: rows_bar {tuple(rows_bar.shape)} does not fit index {tuple(index.shape)}, num_rows {num_rows}")
    d = rows_bar.shape[-1]
    idx, bits = _index(index, rows_bar, "embedding_backward")
    n = idx.numel()
    g2, ldg = _matrix(rows_bar, n, d, rows_bar, "rows_bar")
    out = rows_bar.new_empty((num_rows, d))
    ws, nbytes = _workspace(rows_bar, "nrh_embedding_backward_workspace_bytes", n, num_rows, d)
    with _Here(rows_bar.device) as stream:
        rc = _lib.load().nrh_embedding_backward(dtype, g2.data_ptr(), ldg, idx.data_ptr(), bits, n, num_rows, d, scale, out.data_ptr(), d, _vp(ws),
                                                nbytes, stream)
    _lib.check(rc, "nrh_embedding_backward")
    return out
