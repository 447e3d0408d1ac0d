"""Layer normalisation and the Muon update: the cases they are measured at, their plain forms and their definitions.

Two operators, each with the forms a training or a serving program calls:

* layer normalisation over the last axis (``functional.layer_norm``): forward alone, and forward with the gradients
  of the input, the scale and the offset;
* orthogonalisation of matrices by Newton-Schulz products (``functional.orthogonalize``), and the optimizer step built
  on it (``make_optimizer("muon", ...)``): momentum, orthogonalisation and weight update of a model's matrices.

``run`` computes the plain form, elementary tensor operations in 32 bits, or with ``own`` set calls the framework.
``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
# quintic Newton-Schulz iteration of the Muon optimizer: X <- a X + (b A + c A A) X with A = X X^T
QUINTIC = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-7
STEPS = 5
LR, MOMENTUM, DECAY = 0.02, 0.95, 1e-2

# the convolution and dense kernels of the flower CNN as [outputs, inputs of one output] (first layer: 8-channel
# pixels; last: 5 classes padded to 8 rows)
FLOWER_CNN = "32x72,64x288,128x576,256x1152,512x2304,1024x512,8x1024"
# ... and of ResNet-50, stage by stage (blocks x (reduce, 3x3, expand) + projection, stem, 1000 classes)
RESNET50 = ",".join(
    ["64x392", "64x64"] + ["64x256"] * 2 + ["64x576"] * 3 + ["256x64"] * 4
    + ["128x256"] + ["128x512"] * 3 + ["128x1152"] * 4 + ["512x128"] * 4 + ["512x256"]
    + ["256x512"] + ["256x1024"] * 5 + ["256x2304"] * 6 + ["1024x256"] * 6 + ["1024x512"]
    + ["512x1024"] + ["512x2048"] * 2 + ["512x4608"] * 3 + ["2048x512"] * 3 + ["2048x1024"] + ["1000x2048"])


def listed():
    return [
        # pooled features of one served image
        {"name": "norm_one_row", "op": "norm", "train": False, "rows": 1, "cols": 2048, "pitch": 2048, "type": "bf16"},
        # a branch's channels inside the wider buffer that an Inception block concatenates into, batch 64 at 35 x 35
        {"name": "norm_channel_slice", "op": "norm", "train": False, "rows": 64 * 35 * 35, "cols": 288, "pitch": 768,
         "type": "bf16"},
        # the head's features in a training step at batch 256
        {"name": "norm_train_head", "op": "norm", "train": True, "rows": 256, "cols": 2048, "pitch": 2048, "type": "bf16"},
        # a stage-1 feature map of 256 images, normalised over its 64 channels
        {"name": "norm_train_map", "op": "norm", "train": True, "rows": 256 * 56 * 56, "cols": 64, "pitch": 64,
         "type": "bf16"},
        # odd rows and columns in single precision
        {"name": "norm_train_odd", "op": "norm", "train": True, "rows": 4099, "cols": 1001, "pitch": 1001, "type": "fp32"},
        # long rows, many of them
        {"name": "norm_train_wide", "op": "norm", "train": True, "rows": 16384, "cols": 8192, "pitch": 8192,
         "type": "bf16"},
        # one 3x3 kernel of ResNet-50's first stage
        {"name": "orthogonalize_small", "op": "orthogonalize", "batch": 1, "rows": 64, "cols": 576, "type": "bf16"},
        # the six 3x3 kernels of its third stage at once, single precision
        {"name": "orthogonalize_batch", "op": "orthogonalize", "batch": 6, "rows": 256, "cols": 2304, "type": "fp32"},
        # a tall matrix of odd sizes
        {"name": "orthogonalize_odd", "op": "orthogonalize", "batch": 1, "rows": 1531, "cols": 777, "type": "fp32"},
        # a large square matrix
        {"name": "orthogonalize_large", "op": "orthogonalize", "batch": 1, "rows": 4096, "cols": 4096, "type": "bf16"},
        # optimizer step over every matrix of the flower CNN
        {"name": "muon_flower_cnn", "op": "muon", "shapes": FLOWER_CNN, "nesterov": True, "grad": "fp32"},
        # ... and of ResNet-50
        {"name": "muon_resnet50", "op": "muon", "shapes": RESNET50, "nesterov": True, "grad": "fp32"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "orthogonalize", "orthogonalize", "muon"])
    if kind == "norm":
        cols = _log_uniform(rng, 8, 16384)
        rows = _log_uniform(rng, 1, min(1000000, (1 << 26) // cols))
        if rng.random() < 0.5:
            cols = (cols + 7) // 8 * 8
        pitch = cols if rng.random() < 0.7 else cols + rng.choice([8, 64, 5])
        return {"op": "norm", "train": rng.random() < 0.7, "rows": rows, "cols": cols, "pitch": pitch,
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "orthogonalize":
        rows, cols = _log_uniform(rng, 8, 2500), _log_uniform(rng, 8, 2500)
        batch = rng.randint(1, max(1, min(8, 4000000 // (rows * cols))))
        return {"op": "orthogonalize", "batch": batch, "rows": rows, "cols": cols,
                "type": rng.choice(["bf16", "fp16", "fp32", "fp32"])}
    # a plain convolutional classifier: stages that widen, 3x3 and 1x1 kernels, a dense head
    width, cin, shapes = 8 * rng.randint(2, 12), 8, []
    for _ in range(rng.randint(2, 4)):
        for _ in range(rng.randint(1, 4)):
            k = rng.choice([1, 9])
            shapes.append("%dx%d" % (width, k * cin))
            cin = width
        width = min(768, width * 2)
    shapes.append("%dx%d" % (8 * rng.randint(1, 128), cin))
    return {"op": "muon", "shapes": ",".join(shapes), "nesterov": rng.random() < 0.7, "grad": rng.choice(["fp32", "bf16"])}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _offsets(shapes):
    """Matrices laid out one after the other, each at a multiple of 64 values, and the buffer's length."""
    at, out = 0, []
    for r, c in shapes:
        out.append((at, r, c))
        at += (r * c + 63) // 64 * 64
    return out, at


def _gradient(gen, *shape):
    """Matrices shaped like averaged gradients: a few strong directions that decay, over noise."""
    dev = torch.device("cuda")
    noise = torch.randn(shape, generator=gen, device=dev)
    rank = max(1, min(shape[-2:]) // 8)
    left = torch.randn(shape[:-1] + (rank,), generator=gen, device=dev)
    right = torch.randn(shape[:-2] + (rank, shape[-1]), generator=gen, device=dev)
    decay = torch.arange(1, rank + 1, device=dev, dtype=torch.float32) ** -0.5
    return (noise + (left * decay) @ right) * 1e-3


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = dict(case)
    if case["op"] == "norm":
        dt, rows, cols, pitch = DTYPES[case["type"]], case["rows"], case["cols"], case["pitch"]

        def matrix(scale, shift):
            m = torch.randn(rows, pitch, generator=gen, device=dev).mul_(scale).add_(shift)
            return m.to(dt)[:, :cols]

        state["x"] = matrix(1.5, 0.3)
        state["gamma"] = 1.0 + 0.2 * torch.randn(cols, generator=gen, device=dev)
        state["beta"] = 0.1 * torch.randn(cols, generator=gen, device=dev)
        if case["train"]:
            state["dy"] = matrix(0.01, 0.0)
            for k in ("x", "gamma", "beta"):
                state[k].requires_grad_(True)
        return state
    if case["op"] == "orthogonalize":
        state["x"] = _gradient(gen, case["batch"], case["rows"], case["cols"]).to(DTYPES[case["type"]])
        return state
    places, total = _offsets(_shapes(case))
    state["places"] = places
    for k in ("w", "g", "buf"):
        state[k] = torch.zeros(total, device=dev)
    for at, r, c in places:
        state["w"][at:at + r * c] = torch.randn(r * c, generator=gen, device=dev) * math.sqrt(2.0 / c)
        state["g"][at:at + r * c] = _gradient(gen, r, c).reshape(-1)
        state["buf"][at:at + r * c] = 8.0 * _gradient(gen, r, c).reshape(-1)
    state["g"] = state["g"].to(DTYPES[case["grad"]])
    state["w16"] = state["w"].to(torch.bfloat16)
    if own:
        from distributed_tensorflow_amd.optim import OptRegion, make_optimizer

        region = OptRegion("weights", state["w"], state["g"], state["w16"], True, matrices=places)
        opt = make_optimizer("muon", [region], LR, momentum=MOMENTUM, nesterov=case["nesterov"], weight_decay=DECAY)
        opt.buf["weights"].copy_(state["buf"])
        state["buf"], state["optimizer"] = opt.buf["weights"], opt
    return state


# ------------------------------------------------------------------ plain forms
def _plain_orthogonalize(x):
    """``x [..., r, c]`` in 32 bits; the norm, one long sum, in 64."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    a, b, c = QUINTIC
    norm = x.double().square().sum((-1, -2), keepdim=True).sqrt() + NORM_EPS
    x = (x / norm).float()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2).contiguous() if tall else x


def _plain_norm(s):
    x = s["x"].detach().float()
    gamma, beta = s["gamma"].detach(), s["beta"].detach()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * gamma + beta).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    d = dy * gamma
    dx = rstd * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * hat).sum(0), dy.sum(0)


def _plain_muon(s):
    for at, r, c in s["places"]:
        view = slice(at, at + r * c)
        g, w, buf = s["g"][view].float(), s["w"][view], s["buf"][view]
        buf.mul_(MOMENTUM).add_(g)
        u = g + MOMENTUM * buf if s["nesterov"] else buf
        o = _plain_orthogonalize(u.view(r, c)).reshape(-1)
        w.copy_(w * (1.0 - LR * DECAY) - LR * math.sqrt(max(1.0, r / c)) * o)
        s["w16"][view] = w.to(torch.bfloat16)
    return s["w"], s["w16"], s["buf"]


def run(state):
    op = state["op"]
    if own:
        from distributed_tensorflow_amd.ops import functional as F

        if op == "norm":
            y = F.layer_norm(state["x"], state["gamma"], state["beta"], eps=EPS)
            if not state["train"]:
                return y
            grads = torch.autograd.grad(y, (state["x"], state["gamma"], state["beta"]), state["dy"])
            return (y.detach(),) + grads
        if op == "orthogonalize":
            return F.orthogonalize(state["x"], steps=STEPS)
        state["optimizer"].step()
        return state["w"], state["w16"], state["buf"]
    if op == "norm":
        return _plain_norm(state)
    if op == "orthogonalize":
        return _plain_orthogonalize(state["x"].float()).to(state["x"].dtype)
    return _plain_muon(state)


# ------------------------------------------------------------------ definitions in 64 bits
def _exact_orthogonalize(g):
    a, b, c = QUINTIC
    q = g / (torch.linalg.vector_norm(g) + NORM_EPS)
    wide = q.shape[0] <= q.shape[1]
    for _ in range(STEPS):
        s = q @ q.T if wide else q.T @ q
        p = s @ (s * c)
        p.add_(s, alpha=b)
        p.diagonal().add_(a)
        q = p @ q if wide else q @ p
    return q


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        gamma, beta = s["gamma"].detach().double(), s["beta"].detach().double()
        y = torch.empty(rows, cols, dtype=torch.float64, device="cuda")
        dx = torch.empty_like(y) if case["train"] else None
        dgamma = torch.zeros(cols, dtype=torch.float64, device="cuda")
        dbeta = torch.zeros_like(dgamma)
        step = max(1, (1 << 24) // cols)
        for lo in range(0, rows, step):
            x = s["x"].detach()[lo:lo + step].double()
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            inv = 1.0 / torch.sqrt(var + EPS)
            hat = (x - mean) * inv
            y[lo:lo + step] = torch.addcmul(beta, hat, gamma)
            if case["train"]:
                dy = s["dy"][lo:lo + step].double()
                along = (dy * gamma * hat).sum(1, keepdim=True) / cols
                level = (dy * gamma).sum(1, keepdim=True) / cols
                dx[lo:lo + step] = (dy * gamma - level - along * hat) * inv
                dgamma += (dy * hat).sum(0)
                dbeta += dy.sum(0)
        return (y, dx, dgamma, dbeta) if case["train"] else y
    if case["op"] == "orthogonalize":
        return torch.stack([_exact_orthogonalize(m) for m in s["x"].double()])
    w, g, m = s["w"].double(), s["g"].double(), s["buf"].double()
    m = MOMENTUM * m + g
    u = MOMENTUM * m + g if case["nesterov"] else m
    for at, r, c in s["places"]:
        end = at + r * c
        step = _exact_orthogonalize(u[at:end].view(r, c)) * math.sqrt(max(r, c) / c)
        w[at:end] -= LR * (DECAY * w[at:end] + step.reshape(-1))
    return w, w, m


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["cols"], SIZES[case["type"]]
        if case["train"]:  # x and dy in, y and dx out; scale and offset in, their gradients out
            return {"bytes": 4 * n * size + 16 * case["cols"], "flops": 20 * n}
        return {"bytes": 2 * n * size + 8 * case["cols"], "flops": 8 * n}
    if case["op"] == "orthogonalize":
        shapes, size = [(case["rows"], case["cols"])] * case["batch"], 2 * SIZES[case["type"]]
    else:  # gradient, momentum and weights in; momentum, weights and their bf16 copy out
        shapes, size = _shapes(case), SIZES[case["grad"]] + 4 + 4 + 4 + 4 + 2
    flops = 0
    for r, c in shapes:
        m, n = min(r, c), max(r, c)
        flops += STEPS * (m * m * n + m * m * m + 2 * m * m * n)  # the two symmetric products by half
    return {"bytes": sum(r * c for r, c in shapes) * size, "flops": flops}
