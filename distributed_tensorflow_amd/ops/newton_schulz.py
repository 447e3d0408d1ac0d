"""Orthogonalisation by Newton-Schulz products: plans and launches.

A plan holds, for a list of matrices, their places in a padded workspace and the work lists of every stage, uploaded
once per (shapes, device) -- like a convolution's tap table.  A call allocates its workspace through the caching
allocator, so calls on different streams, and captured graphs, never share one.
"""
from __future__ import annotations

import ctypes as C
import math
from collections import Counter
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import hipk

F32 = torch.float32
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # as in row_io.h
NORM_EPS = 1e-7
MAX_SIDE = 1 << 20        # rows, columns
MAX_SHORT_SIDE = 1 << 15  # the smaller of the two: its square is a plane of the workspace
MAX_STEPS = 12            # what the held bits of small entries carry (newton_schulz.hip)
SCALE = 2.0 ** 15         # of X as it is held: entries of at most 1.21 stay below fp16's 65504
MAX_PARTS = 1024          # partial sums of squares per matrix
CHUNK = 8192              # elements per partial sum, at least
# Workspace of a batch: larger ones go in groups, one after the other (a matrix at least).  A group fills the card many times
# over: with 256 MiB 64 of 1024 x 1024 took 5.66 instead of 5.29 ms, 40 of 64 x 8192 0.52 instead of 0.43.
GROUP_BYTES = 2 << 30

# Measured on one MI355X, a CU's time in us: a tile job's fixed part (its first loads, the epilogue) and a k-step of 32.
# A 128 x 128 tile does four times the work of a 64 x 64 tile in twice the time, so large tiles win once there are enough
# of them for 256 CUs.
JOB_US = {128: 5.0, 64: 1.5}
STEP_US = {128: 0.72, 64: 0.31}
JOIN_US, JOIN_US_PER_BYTE = 4.0, 0.25e-6   # the launch that joins cut reductions (8 MB of slabs 6 us, 127 MB 36 us)
CUS = 256
SLOTS = 2 * CUS           # workgroups at a time
MIN_STEPS = 8             # least upper bound of the pieces of a cut reduction (cut evenly: 9 k-steps make pieces of 4 and 5)

# Shorter sides of at most 64 take one launch an iteration, in which every workgroup adds up the partial products of all
# slices of its matrix (about 0.25 us each) and advances the 64 x 64 blocks of its own (about 2.5 us each): the time is
# least at sqrt(10 * blocks) slices.  64 x 576 bf16: 46 us against 80 in separate stages, 64 x 4608: 81 against 108.
SMALL_BLOCKS_PER_SLICE2 = 10.0
SMALL_MAX_LONG = 8192

_MAT = np.dtype([("at", "<i8"), ("x", "<i8"), ("a", "<i8"), ("part", "<i8"), ("rows", "<i4"), ("cols", "<i4"),
                 ("rp", "<i4"), ("cp", "<i4"), ("mp", "<i4"), ("parts", "<i4"), ("chunk", "<i4"), ("tall", "<i4"),
                 ("scale", "<f4"), ("lr_scale", "<f4")])   # NsMat


class NsArgs(C.Structure):
    _fields_ = [("mats", C.c_void_p), ("chunks", C.c_void_p), ("packs", C.c_void_p), ("gram", C.c_void_p),
                ("joins", C.c_void_p), ("poly", C.c_void_p), ("poly_joins", C.c_void_p), ("full", C.c_void_p),
                ("small", C.c_void_p), ("nsmall", C.c_int), ("small_slices", C.c_int), ("nchunks", C.c_int),
                ("npacks", C.c_int), ("ngram", C.c_int), ("ngram_joins", C.c_int), ("npoly", C.c_int), ("npoly_joins", C.c_int),
                ("nfull", C.c_int), ("steps", C.c_int), ("dtype", C.c_int), ("large", C.c_int),
                ("in_", C.c_void_p), ("out", C.c_void_p), ("buf", C.c_void_p), ("w", C.c_void_p), ("w16", C.c_void_p),
                ("hyper", C.c_void_p), ("part", C.c_void_p), ("slabs", C.c_void_p), ("ws", C.c_void_p), ("nparts", C.c_longlong),
                ("eps", C.c_float), ("mu", C.c_float), ("wd", C.c_float), ("nesterov", C.c_int)]


def check_shape(rows: int, cols: int, what: str) -> None:
    if rows < 1 or cols < 1:
        raise ValueError("%s: a matrix needs at least one row and one column, got %d x %d" % (what, rows, cols))
    if max(rows, cols) > MAX_SIDE or min(rows, cols) > MAX_SHORT_SIDE:
        raise ValueError("%s: %d x %d is too large (at most 2^20, the smaller side at most 2^15)" % (what, rows, cols))


def _tiles(rows: int, cols: int, lower: bool = False) -> Tuple[np.ndarray, np.ndarray]:
    """Rows and columns of every tile of a grid, or of those on and below the diagonal, block by block of 8 x 8."""
    i, j = np.divmod(np.arange(rows * cols, dtype=np.int64), cols)
    if lower:
        i, j = i[j <= i], j[j <= i]
    order = np.lexsort((j, i, j // 8, i // 8))
    return i[order], j[order]


def _jobs(mat: int, i, j, edge: int, k0, k1, slab=-1) -> np.ndarray:
    """NsJob records {matrix, tile row, tile column, edge, k0, k1, slab, -}."""
    out = np.zeros((len(i), 8), dtype=np.int32)
    for c, v in enumerate((mat, i, j, edge, k0, k1, slab)):
        out[:, c] = v
    return out


def _job_us(edge: int, steps: float) -> float:
    return JOB_US[edge] + STEP_US[edge] * steps


def _cost(jobs: np.ndarray) -> np.ndarray:
    large = jobs[:, 3] == 128
    return (np.where(large, JOB_US[128], JOB_US[64])
            + np.where(large, STEP_US[128], STEP_US[64]) * ((jobs[:, 5] - jobs[:, 4]) // 32))


def _up(v: int, edge: int) -> int:
    return -(-v // edge) * edge


def _span(jobs: Sequence[Tuple[int, float]]) -> float:
    """Time of a launch of (count, cost) jobs, longest first.  Two workgroups share a CU's matrix cores, so what counts is
    the work per CU, or what the CU with the most of the longest jobs takes; and a long job that started first has had half
    a CU for as long as there were others to start.  (ResNet-50's A stage in 35 cuttings, 55 .. 130 us: within 15 % of the
    measured times; without the last term the best by estimate took 84 us where the best takes 67.)"""
    span = count = total = longest = 0.0
    for n, cost in sorted(jobs, key=lambda j: -j[1]):
        longest = longest or cost
        count += n
        total += n * cost
        span = max(span, math.ceil(count / CUS) * cost)
    share = total / CUS
    return max(span, share * 1.08, longest + share / 2 if count > 0.9 * CUS else 0.0)


def _choose(dims: Sequence[Tuple[int, int, int]], symmetric: bool) -> Tuple[int, int]:
    """(size of the shorter of tile rows / columns from which tiles are 128, longest piece of a reduction in k-steps) of a
    stage whose outputs are ``rows x cols`` sums over ``K`` for (rows, cols, K) in ``dims``."""
    best: Optional[Tuple[float, int, int]] = None
    alike = Counter(dims)
    for large_from in (128, 256, 512, 1024, 1 << 30):
        for piece in (1 << 30, 64, 48, 40, 32, 28, 24, 20, 16, 12, MIN_STEPS) if symmetric else (1 << 30,):
            jobs: Dict[float, int] = {}
            slabs = 0
            for (rows, cols, K), many in alike.items():
                edge = 128 if min(rows, cols) >= large_from else 64
                tr, tc, steps = -(-rows // edge), -(-cols // edge), _up(K, edge) // 32
                n = (tr * (tr + 1) // 2 if symmetric else tr * tc) * many
                cut = -(-steps // piece)
                cost = _job_us(edge, -(-steps // cut))
                jobs[cost] = jobs.get(cost, 0) + n * cut
                slabs += n * cut * edge * edge * 4 if cut > 1 else 0
            if symmetric and len(dims) == 1 and cut == 1 and _tail(n):   # (the tail's work is spread by _cut_tail)
                jobs[cost] = n - _tail(n)
                jobs[cost * _tail(n) / CUS] = CUS
                slabs = SLOTS * edge * edge * 4
            time = _span([(n, cost) for cost, n in jobs.items()]) + (JOIN_US + slabs * JOIN_US_PER_BYTE if slabs else 0.0)
            if best is None or time < best[0]:
                best = (time, large_from, piece)
    return best[1], best[2]


def _cut(jobs: np.ndarray, piece: int, slabs: int) -> Tuple[np.ndarray, np.ndarray, int]:
    """Jobs with their reductions cut into pieces of at most ``piece`` k-steps, the jobs that join the slabs of those that
    were, and the next free slab."""
    steps = int(jobs[0, 5] - jobs[0, 4]) // 32
    cut = -(-steps // piece)
    if cut == 1:
        return jobs, jobs[:0], slabs
    unit = (int(jobs[0, 3]) // 64) ** 2
    out = np.repeat(jobs, cut, axis=0)
    at = np.tile(np.arange(cut), len(jobs))
    out[:, 4], out[:, 5] = at * steps // cut * 32, (at + 1) * steps // cut * 32
    out[:, 6] = slabs + np.arange(len(out)) * unit
    joins = jobs.copy()
    joins[:, 4], joins[:, 6] = cut, slabs + np.arange(len(jobs)) * cut * unit
    return out, joins, slabs + len(out) * unit


def _tail(n: int) -> int:
    """How many of ``n`` equal jobs lie beyond whole rounds of workgroups and would run on a mostly idle card."""
    tail = n % SLOTS
    return tail if n >= SLOTS and tail <= SLOTS // 2 else 0


def _cut_tail(jobs: np.ndarray, slabs: int) -> Tuple[np.ndarray, np.ndarray, int]:
    """The reductions of such jobs are cut so that the whole card takes part."""
    tail = _tail(len(jobs))
    if not tail:
        return jobs, jobs[:0], slabs
    steps = int(jobs[0, 5] - jobs[0, 4]) // 32
    piece = max(MIN_STEPS, -(-steps // max(2, SLOTS // tail)))
    cut, joins, slabs = _cut(jobs[-tail:], piece, slabs)
    return np.concatenate([jobs[:-tail], cut]), joins, slabs


def _repeat(jobs: np.ndarray, n: int, mat: int, slab: int = 0, slabs: int = 0) -> np.ndarray:
    """The jobs of one matrix for ``n`` alike from number ``mat`` on, whose slabs follow one another from ``slab`` on,
    ``slabs`` for each."""
    out = np.tile(jobs, (n, 1))
    which = np.repeat(np.arange(n, dtype=np.int32), len(jobs))
    out[:, 0] = mat + which
    if jobs.shape[1] == 8:
        out[:, 6] = np.where(out[:, 6] >= 0, out[:, 6] + slab + which * slabs, out[:, 6])
    return out


def _join(parts: Sequence[np.ndarray], width: int = 8) -> np.ndarray:
    return np.concatenate(parts) if parts else np.zeros((0, width), dtype=np.int32)


def _over_xcds(groups: Sequence[np.ndarray]) -> np.ndarray:
    """Workgroup n runs on XCD n % 8, each with its own L2: neighbouring tiles, which read the same rows, go to the same
    XCD.  Every run of equal jobs is dealt out in eight consecutive parts, what does not divide job by job to the XCDs
    with the least work so far; within an XCD the longest jobs start first.  Shorter queues end in empty jobs."""
    if not groups:
        return _join(groups)
    runs = []
    for g in groups:
        runs += np.split(g, np.flatnonzero(np.diff(_cost(g))) + 1)
    runs.sort(key=lambda g: -float(_cost(g[:1])[0]))
    queues: List[List[np.ndarray]] = [[] for _ in range(8)]
    load = np.zeros(8)
    for g in runs:
        each, cost = len(g) // 8, float(_cost(g[:1])[0])
        for x in range(8):
            queues[x].append(g[x * each:(x + 1) * each])
        load += each * cost
        for n in range(8 * each, len(g)):
            x = int(np.argmin(load))
            queues[x].append(g[n:n + 1])
            load[x] += cost
    longest = max(sum(len(g) for g in q) for q in queues)
    out = np.zeros((longest, 8, 8), dtype=np.int32)
    out[:, :, 0] = -1
    for x, q in enumerate(queues):
        jobs = np.concatenate(q)
        out[:len(jobs), x] = jobs[np.argsort(-_cost(jobs), kind="stable")]
    out = out.reshape(-1, 8)
    return out[:len(out) - int(np.argmax(out[::-1, 0] >= 0))]   # (no empty jobs behind the last)


class NsPlan:
    """Places and work lists of ``matrices`` (offset, rows, cols), each contiguous at its offset."""

    def __init__(self, matrices: Sequence[Tuple[int, int, int]], device):
        mats = np.zeros(len(matrices), dtype=_MAT)
        for _, rows, cols in matrices:
            check_shape(rows, cols, "orthogonalize")
        sides = [(min(rows, cols), max(rows, cols)) for _, rows, cols in matrices]
        fused = max(short for short, _ in sides) <= 64 and max(long for _, long in sides) <= SMALL_MAX_LONG
        gram_large, gram_piece = _choose([(short, short, long) for short, long in sides], True)
        poly_large, poly_piece = _choose([(short, short, short) for short, _ in sides], True)
        full_large, _ = _choose([(short, long, short) for short, long in sides], False)
        chunks, packs, gram, gram_joins, poly, poly_joins, full = [], [], [], [], [], [], []
        small: List[np.ndarray] = []
        ws = part = gram_slabs = poly_slabs = small_slices = 0
        k = 0
        while k < len(matrices):   # runs of matrices of one shape
            _, rows, cols = matrices[k]
            many = 1
            while k + many < len(matrices) and tuple(matrices[k + many][1:]) == (rows, cols):
                many += 1
            short = min(rows, cols)
            edge = 128 if short >= min(gram_large, poly_large, full_large) else 64
            rp, cp, mp = _up(rows, edge), _up(cols, edge), _up(short, edge)
            n = rows * cols
            chunk = max(CHUNK, _up(-(-n // MAX_PARTS), CHUNK))
            parts = -(-n // chunk)
            elems = 4 * rp * cp + 4 * mp * mp
            run = mats[k:k + many]
            run["at"] = [at for at, _, _ in matrices[k:k + many]]
            run["x"] = ws + np.arange(many, dtype=np.int64) * elems
            run["a"] = run["x"] + 4 * rp * cp
            run["part"] = part + np.arange(many, dtype=np.int64) * parts
            for name, v in (("rows", rows), ("cols", cols), ("rp", rp), ("cp", cp), ("mp", mp), ("parts", parts),
                            ("chunk", chunk), ("tall", rows > cols), ("scale", SCALE),
                            ("lr_scale", math.sqrt(max(1.0, rows / cols)))):
                run[name] = v
            ws += many * elems
            part += many * parts
            i = np.arange(parts, dtype=np.int32)
            chunks.append(_repeat(np.stack([0 * i, i, 0 * i, 0 * i], 1), many, k))
            if fused:
                blocks = max(rp, cp) // 64
                slices = min(blocks, max(1, round(math.sqrt(SMALL_BLOCKS_PER_SLICE2 * blocks))))
                edges = np.arange(slices + 1) * blocks // slices
                jobs = _jobs(0, np.arange(slices), edges[:-1], np.diff(edges), slices, 0, 0)
                small.append(_repeat(jobs, many, k, small_slices, slices))
                small_slices += many * slices
                k += many
                continue
            i, j = _tiles(rp // 64, cp // 64)
            packs.append(_repeat(np.stack([0 * i, i, j, 0 * i], 1).astype(np.int32), many, k))
            e = 128 if short >= gram_large else 64
            jobs, joins, used = _cut(_jobs(0, *_tiles(mp // e, mp // e, lower=True), e, 0, max(rp, cp)), gram_piece, 0)
            if len(matrices) == 1 and not len(joins):
                jobs, joins, used = _cut_tail(jobs, 0)
            gram += np.split(_repeat(jobs, many, k, gram_slabs, used), many)
            gram_joins.append(_repeat(joins, many, k, gram_slabs, used))
            gram_slabs += many * used
            e = 128 if short >= poly_large else 64
            jobs, joins, used = _cut(_jobs(0, *_tiles(mp // e, mp // e, lower=True), e, 0, mp), poly_piece, 0)
            if len(matrices) == 1 and not len(joins):
                jobs, joins, used = _cut_tail(jobs, 0)
            poly += np.split(_repeat(jobs, many, k, poly_slabs, used), many)
            poly_joins.append(_repeat(joins, many, k, poly_slabs, used))
            poly_slabs += many * used
            e = 128 if short >= full_large else 64
            full += np.split(_repeat(_jobs(0, *_tiles(rp // e, cp // e), e, 0, mp), many, k), many)
            k += many
        if fused:   # one launch an iteration
            gram_slabs = 2 * small_slices
        slabs = max(gram_slabs, poly_slabs)   # (a stage's slabs are joined before the next stage writes its own)
        lists = [np.concatenate(chunks), _join(packs, 4), _over_xcds(gram), _join(gram_joins), _over_xcds(poly),
                 _join(poly_joins), _over_xcds(full), _join(small)]
        counts = [len(v) for v in lists]
        self.counts = [counts[7], small_slices] + counts[:7]
        self.large = sum(bit for bit, at in ((1, 2), (2, 4), (4, 6)) if (lists[at][:, 3] == 128).any())
        # 32-byte aligned: the lists are read 16 and 32 bytes at a time
        blobs = [v.tobytes() + b"\0" * (-v.nbytes % 32) for v in [mats] + lists]
        self.table = torch.from_numpy(np.frombuffer(b"".join(blobs), dtype=np.uint8).copy()).to(device)
        starts = np.cumsum([0] + [len(v) for v in blobs])
        self.places = [self.table.data_ptr() + int(s) for s in starts[:9]]
        self.ws_elems, self.parts, self.mats, self.slabs = ws, part, len(matrices), slabs
        self.first = min(at for at, _, _ in matrices)
        self.end = max(at + rows * cols for at, rows, cols in matrices)

    def launch(self, *, inp: torch.Tensor, steps: int, out=None, buf=None, w=None, w16=None, hyper=None, mu=0.0,
               nesterov=False, wd=0.0) -> None:
        dev = inp.device
        if dev != self.table.device:
            raise ValueError("orthogonalize: a plan for %s cannot run on %s" % (self.table.device, dev))
        if self.first < 0 or self.end > inp.numel():
            raise ValueError("orthogonalize: the plan's matrices take the values %d .. %d of a buffer of %d"
                             % (self.first, self.end, inp.numel()))
        with hipk.device_of(inp):
            ws = torch.empty(self.ws_elems, dtype=torch.float16, device=dev)
            part = torch.empty(self.parts + self.mats, dtype=torch.float64, device=dev)
            slabs = torch.empty(self.slabs * 4096, dtype=F32, device=dev) if self.slabs else None
            args = NsArgs(*self.places, *self.counts, steps, DTYPES[inp.dtype], self.large, inp.data_ptr(), hipk.ptr(out),
                          hipk.ptr(buf), hipk.ptr(w), hipk.ptr(w16), hipk.ptr(hyper), part.data_ptr(), hipk.ptr(slabs), ws.data_ptr(),
                          self.parts, NORM_EPS, mu, wd, 1 if nesterov else 0)
            hipk.check(hipk.lib().dtfa_newton_schulz(C.byref(args), hipk.stream()), "newton_schulz")


_plans: Dict[tuple, NsPlan] = {}


def get_plan(key: tuple, matrices: Callable[[], Sequence[Tuple[int, int, int]]], device: torch.device) -> NsPlan:
    """The plan of the matrices that ``key`` stands for on ``device``.  Plans stay for the life of the process, like those of
    the convolutions: kernels in flight on any stream, and captured graphs, hold their addresses."""
    plan = _plans.get((key, device.index))
    if plan is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("orthogonalize: the first call of these shapes uploads their plan and cannot be captured: run "
                               "it once before the capture")
        plan = _plans.setdefault((key, device.index), NsPlan(matrices(), device))
    return plan


def _group(rows: int, cols: int) -> int:
    """How many matrices of a batch go together at most: what GROUP_BYTES hold of their planes, padded to tiles, and slabs."""
    short, long = sorted((rows, cols))
    edge = 64 if short <= 64 else 128
    m, n = _up(short, edge), _up(long, edge)
    slabs = 2 * (n // 64) * 4096 * 4 if short <= 64 else m * m * 4
    return max(1, GROUP_BYTES // (8 * (m * n + m * m) + slabs))


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
    n = rows * cols
    batch = x.numel() // n
    groups = -(-batch // _group(rows, cols))
    for k in range(groups):
        first = k * batch // groups
        many = (k + 1) * batch // groups - first
        plan = get_plan((many, rows, cols), lambda: [(i * n, rows, cols) for i in range(many)], x.device)
        part = slice(first * n, (first + many) * n)
        plan.launch(inp=x.view(-1)[part], steps=steps, out=out.view(-1)[part])
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
    if any(t is not None and t.device != w.device for t in (buf, g, w16, hyper)):
        raise ValueError("muon_step: buffers on different devices")
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError("muon_step: steps must be from 1 to %d, got %r" % (MAX_STEPS, steps))
    plan.launch(inp=g, steps=steps, buf=buf, w=w, w16=w16, hyper=hyper, mu=float(mu), wd=float(wd), nesterov=nesterov)
