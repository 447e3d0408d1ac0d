"""Orthogonalisation by Newton-Schulz products: plans and launches.

A plan holds, for a list of matrices, their places in a padded workspace and the work lists of every stage, uploaded
once per (shapes, device) -- like a convolution's tap table.  A call allocates its workspace through the caching
allocator, so calls on different streams, and captured graphs, never share one.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Dict, Optional, Sequence, Tuple

import numpy as np
import torch

from . import hipk

F32 = torch.float32
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # as in row_io.h
NORM_EPS = 1e-7
MAX_SIDE = 1 << 20        # rows, columns
MAX_SHORT_SIDE = 1 << 15  # the smaller of the two: its square is a plane of the workspace
MAX_STEPS = 64
MAX_PARTS = 1024          # partial sums of squares per matrix
CHUNK = 8192              # elements per partial sum, at least

# edge of the product tiles: 128 from this size of the smaller side on, 64 below
LARGE_TILE_FROM = 512

_MAT = np.dtype([("at", "<i8"), ("x", "<i8"), ("a", "<i8"), ("part", "<i8"), ("rows", "<i4"), ("cols", "<i4"),
                 ("rp", "<i4"), ("cp", "<i4"), ("mp", "<i4"), ("parts", "<i4"), ("chunk", "<i4"), ("tall", "<i4"),
                 ("scale", "<f4"), ("lr_scale", "<f4")])   # NsMat


class NsArgs(C.Structure):
    _fields_ = [("mats", C.c_void_p), ("chunks", C.c_void_p), ("packs", C.c_void_p), ("sym", C.c_void_p), ("full", C.c_void_p),
                ("nchunks", C.c_int), ("npacks", C.c_int), ("nsym", C.c_int), ("nfull", C.c_int),
                ("steps", C.c_int), ("dtype", C.c_int), ("in_", C.c_void_p), ("out", C.c_void_p), ("buf", C.c_void_p),
                ("w", C.c_void_p), ("w16", C.c_void_p), ("hyper", C.c_void_p), ("part", C.c_void_p), ("ws", C.c_void_p), ("nparts", C.c_longlong),
                ("eps", C.c_float), ("mu", C.c_float), ("wd", C.c_float), ("nesterov", C.c_int)]


def check_shape(rows: int, cols: int, what: str) -> None:
    if rows < 1 or cols < 1:
        raise ValueError("%s: a matrix needs at least one row and one column, got %d x %d" % (what, rows, cols))
    if max(rows, cols) > MAX_SIDE or min(rows, cols) > MAX_SHORT_SIDE:
        raise ValueError("%s: %d x %d is too large (at most 2^20, the smaller side at most 2^15)" % (what, rows, cols))


def _tiles(mat: int, rows: int, cols: int, edge: int, lower: bool = False) -> np.ndarray:
    """{matrix, tile row, tile column, edge} of every tile, or of those on and below the diagonal."""
    i, j = np.divmod(np.arange(rows * cols, dtype=np.int64), cols)
    if lower:
        keep = j <= i
        i, j = i[keep], j[keep]
    return np.stack([np.full_like(i, mat), i, j, np.full_like(i, edge)], 1).astype(np.int32)


class NsPlan:
    """Places and work lists of ``matrices`` (offset, rows, cols), each contiguous at its offset."""

    def __init__(self, matrices: Sequence[Tuple[int, int, int]], device):
        mats = np.zeros(len(matrices), dtype=_MAT)
        chunks, packs, sym, full = [], [], [], []
        ws = part = 0
        for k, (at, rows, cols) in enumerate(matrices):
            check_shape(rows, cols, "orthogonalize")
            short = min(rows, cols)
            edge = 128 if short >= LARGE_TILE_FROM else 64
            up = lambda v: -(-v // edge) * edge  # noqa: E731
            rp, cp, mp = up(rows), up(cols), up(short)
            n = rows * cols
            chunk = max(CHUNK, -(-n // (MAX_PARTS * CHUNK)) * CHUNK)
            parts = -(-n // chunk)
            scale = 2.0 ** math.floor(math.log2(min(math.sqrt(n), 2.0 ** 15)))
            mats[k] = (at, ws, ws + 4 * rp * cp, part, rows, cols, rp, cp, mp, parts, chunk, rows > cols, scale,
                       math.sqrt(max(1.0, rows / cols)))
            ws += 4 * rp * cp + 4 * mp * mp
            part += parts
            chunks.append(np.stack([np.full(parts, k), np.arange(parts), np.zeros(parts), np.zeros(parts)], 1).astype(np.int32))
            packs.append(_tiles(k, rp // 64, cp // 64, 64))
            long = max(rp, cp)
            sym.append((-long * edge * edge, _tiles(k, mp // edge, mp // edge, edge, lower=True)))
            full.append((-mp * edge * edge, _tiles(k, rp // edge, cp // edge, edge)))
        # longest tiles first: the last workgroups to start are the short ones
        sym.sort(key=lambda e: e[0])
        full.sort(key=lambda e: e[0])
        lists = [np.concatenate(v) for v in (chunks, packs, [t for _, t in sym], [t for _, t in full])]
        self.counts = [len(v) for v in lists]
        head = mats.tobytes()
        head += b"\0" * (-len(head) % 16)   # the lists are read 16 bytes at a time
        blob = b"".join([head] + [v.tobytes() for v in lists])
        host = torch.from_numpy(np.frombuffer(blob, dtype=np.uint8).copy())
        self.table = host.to(device)
        starts = np.cumsum([0, len(head)] + [v.nbytes for v in lists])
        self.places = [self.table.data_ptr() + int(s) for s in starts[:5]]
        self.ws_elems, self.parts, self.mats = ws, part, len(matrices)

    def launch(self, *, inp: torch.Tensor, steps: int, out=None, buf=None, w=None, w16=None, hyper=None, mu=0.0,
               nesterov=False, wd=0.0) -> None:
        dev = inp.device
        with hipk.device_of(inp):
            ws = torch.empty(self.ws_elems, dtype=torch.float16, device=dev)
            part = torch.empty(self.parts + self.mats, dtype=torch.float64, device=dev)
            args = NsArgs(*self.places, *self.counts, steps, DTYPES[inp.dtype], inp.data_ptr(), hipk.ptr(out), hipk.ptr(buf),
                          hipk.ptr(w), hipk.ptr(w16), hipk.ptr(hyper), part.data_ptr(), ws.data_ptr(),
                          self.parts, NORM_EPS, mu, wd,
                          1 if nesterov else 0)
            hipk.check(hipk.lib().dtfa_newton_schulz(C.byref(args), hipk.stream()), "newton_schulz")


_plans: Dict[tuple, NsPlan] = {}


def get_plan(matrices: Sequence[Tuple[int, int, int]], device: torch.device) -> NsPlan:
    """The plan of these matrices on ``device``.  Plans stay for the life of the process, like those of the convolutions:
    kernels in flight on any stream, and captured graphs, hold their addresses."""
    key = (tuple(matrices), device.index)
    plan = _plans.get(key)
    if plan is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("orthogonalize: the first call of these shapes uploads their plan and cannot be captured: run "
                               "it once before the capture")
        plan = _plans[key] = NsPlan(matrices, device)
    return plan


def orthogonalize(x: torch.Tensor, steps: int) -> torch.Tensor:
    """``x [..., rows, cols]`` on the GPU -> the same shape and dtype (bf16, fp16 or fp32), contiguous."""
    if not x.is_cuda:
        raise ValueError("orthogonalize: x must be a GPU tensor")
    if x.dtype not in DTYPES:
        raise ValueError("orthogonalize: x must be bfloat16, float16 or float32, got %s" % x.dtype)
    rows, cols = x.shape[-2:]
    x = x.contiguous()
    out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    batch = x.numel() // (rows * cols)
    plan = get_plan(tuple((i * rows * cols, rows, cols) for i in range(batch)), x.device)
    plan.launch(inp=x, steps=steps, out=out)
    return out


def muon_step(plan: NsPlan, w: torch.Tensor, buf: torch.Tensor, g: torch.Tensor, w16: Optional[torch.Tensor],
              hyper: torch.Tensor, mu: float, wd: float, nesterov: bool, steps: int) -> None:
    """One Muon step on the matrices of ``plan`` inside the flat buffers ``w``, ``buf`` (fp32), ``g`` (fp32 or bf16) and ``w16``
    (bf16 or None); ``hyper`` = (step size, gradient scale) on the device."""
    for t, nm in ((w, "w"), (buf, "buf"), (hyper, "hyper")):
        hipk.require(t, F32, "muon_step: " + nm)
    n = w.numel()
    if g.dtype not in (F32, torch.bfloat16):
        raise ValueError("muon_step: the gradient must be float32 or bfloat16, got %s" % g.dtype)
    hipk.require(g, g.dtype, "muon_step: gradient")
    if w16 is not None:
        hipk.require(w16, torch.bfloat16, "muon_step: w16")
    if buf.numel() != n or g.numel() != n or (w16 is not None and w16.numel() != n) or hyper.numel() != 2:
        raise ValueError("muon_step: buffer sizes differ")
    plan.launch(inp=g, steps=steps, buf=buf, w=w, w16=w16, hyper=hyper, mu=float(mu), wd=float(wd), nesterov=nesterov)
