"""Operators of a language model's training step, as measurable cases.

  layernorm   layer normalisation over the channels of every position, forward or backward
  fcloss      a fully connected prediction layer over many classes with the softmax loss behind it, whose predictions are
              never stored: forward (loss and log-sum-exp per image) or backward (derivatives of data, filters and biases)
  muon        the trainer's update with the Muon solver: momentum whose matrix is orthogonalised by Newton-Schulz products

Tensors are single precision in MATLAB order H x W x C x N, the first index fastest.  A sequence of tokens is a batch of
1 x 1 x C images; a filter bank FH x FW x FC x K is a matrix of K rows.  ``run`` computes the operators by elementary torch
operations, or through the framework where ``own`` is true.
"""
import math

import torch

own = False

# Filter banks of VGG-16 without their biases, FH x FW x FC x K
_VGG16 = ((3, 3, 3, 64), (3, 3, 64, 64), (3, 3, 64, 128), (3, 3, 128, 128), (3, 3, 128, 256), (3, 3, 256, 256), (3, 3, 256, 256),
          (3, 3, 256, 512), (3, 3, 512, 512), (3, 3, 512, 512), (3, 3, 512, 512), (3, 3, 512, 512), (3, 3, 512, 512),
          (7, 7, 512, 4096), (1, 1, 4096, 4096), (1, 1, 4096, 1000))

_EPSILON = 1e-5                                     # layer normalisation
_MUON = dict(momentum=0.95, nesterov=True, steps=5, a=3.4445, b=-4.7750, c=2.0315, epsilon=1e-7)
_GRAD_MULT, _DECAY, _RATE = 0.5, 5e-4, 0.02


def listed():
    ln = lambda name, back, h, w, c, n: dict(name=name, op="layernorm", back=back, h=h, w=w, c=c, n=n)              # noqa: E731
    fc = lambda name, back, n, d, k: dict(name=name, op="fcloss", back=back, n=n, d=d, k=k)                          # noqa: E731
    mu = lambda name, bank, fs, fc, k, count: dict(name=name, op="muon", bank=bank, fs=fs, fc=fc, k=k, count=count)  # noqa: E731
    return [
        # one token through a layer, as when a sequence is produced step by step: latency alone counts
        ln("ln_one_token", False, 1, 1, 1024, 1),
        # channels of feature maps between convolutions, a batch of images: strided rows
        ln("ln_maps_28x28x512_b64", False, 28, 28, 512, 64),
        # the backward pass over the tokens of a large training batch
        ln("ln_back_16384x4096", True, 1, 1, 4096, 16384),
        # odd maps and channels, backward
        ln("ln_back_maps_35x47x90_b9", True, 35, 47, 90, 9),
        # one token scored against a large vocabulary
        fc("fcloss_one_token_32000", False, 1, 1024, 32000),
        # the last layer of an image classifier of 1000 classes
        fc("fcloss_back_classifier_b64", True, 64, 4096, 1000),
        # a training batch of tokens over a large vocabulary, odd sizes: backward
        fc("fcloss_back_2047x1000x50001", True, 2047, 1000, 50001),
        # the loss of a large batch over a very large vocabulary
        fc("fcloss_8192x2048x100000", False, 8192, 2048, 100000),
        # one convolution's filter bank
        mu("muon_conv_3x3x64x64", "", 3, 64, 64, 1),
        # the square matrices of four layers, one call
        mu("muon_4x_2048x2048", "", 1, 2048, 2048, 4),
        # a bank with more filters than inputs, odd sizes
        mu("muon_1x1x129x1000", "", 1, 129, 1000, 1),
        # every filter bank of VGG-16 in one call
        mu("muon_vgg16", "vgg16", 0, 0, 0, 1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("layernorm", "fcloss", "muon"))
    if op == "layernorm":
        while True:
            case = dict(op=op, back=rng.random() < 0.5, h=1, w=1, c=_log(rng, 16, 8192), n=_log(rng, 1, 16384))
            if rng.random() < 0.5:
                case.update(h=_log(rng, 2, 64), w=_log(rng, 2, 64), c=_log(rng, 16, 1024), n=_log(rng, 1, 64))
            if case["h"] * case["w"] * case["c"] * case["n"] <= 16384 * 4096:
                return case
    if op == "fcloss":
        while True:
            case = dict(op=op, back=rng.random() < 0.5, n=_log(rng, 1, 8192), d=_log(rng, 16, 4096), k=_log(rng, 10, 131072))
            if case["n"] * case["d"] * case["k"] * (3 if case["back"] else 1) <= 8192 * 2048 * 100000:
                return case
    while True:
        fs = rng.choice((1, 1, 3))
        case = dict(op=op, bank="", fs=fs, fc=_log(rng, 8, 4096 // (fs * fs)), k=_log(rng, 8, 4096), count=rng.randint(1, 6))
        if sum(_muon_flops(case)) <= sum(_muon_flops(dict(bank="vgg16"))):
            return case


def _shapes(case):
    return list(_VGG16) if case["bank"] == "vgg16" else [(case["fs"], case["fs"], case["fc"], case["k"])] * case["count"]


def _muon_flops(case):
    out = []
    for fh, fw, fc, k in _shapes(case):
        m, n = sorted((fh * fw * fc, k))
        out.append(_MUON["steps"] * (m * m * n + m * m * m + 2 * m * m * n))     # A and A^2 are symmetric: half of each
    return out


def work(case):
    if case["op"] == "layernorm":
        e, c = case["h"] * case["w"] * case["c"] * case["n"], case["c"]
        return {"bytes": 4 * (3 * e + 3 * c) if case["back"] else 4 * (2 * e + 2 * c), "flops": (14 if case["back"] else 8) * e}
    if case["op"] == "fcloss":
        n, d, k = case["n"], case["d"], case["k"]
        tensors = n * d + k * d + k
        return {"bytes": 4 * (2 * tensors + 2 * n) if case["back"] else 4 * (tensors + 2 * n), "flops": (6 if case["back"] else 2) * n * d * k}
    size = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 4 * 5 * size, "flops": sum(_muon_flops(case))}               # W and momentum read and written, gradient read


# ------------------------------------------------------------------------------------------------------- inputs
def _tensor(gen, shape, std=1.0, mean=0.0):
    """Normal values in column-major order."""
    t = torch.empty(tuple(reversed(shape)), device="cuda").normal_(mean, std, generator=gen)
    return t.permute(tuple(range(len(shape) - 1, -1, -1)))


def _rows(t):
    """A column-major tensor as a row-major matrix with one row per index of its last dimension."""
    return t.permute(tuple(range(t.dim() - 1, -1, -1))).reshape(t.shape[-1], -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "layernorm":
        shape = (case["h"], case["w"], case["c"], case["n"])
        scale = torch.empty(case["c"], device="cuda").uniform_(0.5, 2.0, generator=gen)      # channels differ in size
        x = (_rows(_tensor(gen, shape, 1.0, 0.3)).view(case["n"], case["c"], -1) * scale[None, :, None])
        x = x.view(tuple(reversed(shape))).permute(3, 2, 1, 0)
        g, b = _tensor(gen, (case["c"], 1), 0.2, 1.0), _tensor(gen, (case["c"], 1), 0.2)
        return dict(case, x=x, g=g, bias=b, dzdy=_tensor(gen, shape) if case["back"] else None)
    if case["op"] == "fcloss":
        n, d, k = case["n"], case["d"], case["k"]
        x, f, b = _tensor(gen, (1, 1, d, n)), _tensor(gen, (1, 1, d, k), 1.5 / math.sqrt(d)), _tensor(gen, (k, 1), 0.5)
        labels = torch.randint(1, k + 1, (n,), device="cuda", generator=gen).float()
        if n > 8:                                                                            # padding: images without a class
            labels[torch.rand(n, device="cuda", generator=gen) < 0.05] = 0.0
        lse = _logits_lse(_rows(x), _rows(f), b.reshape(-1), labels) if case["back"] else None   # kept from the forward pass
        return dict(case, x=x, f=f, bias=b, labels=labels, lse=lse)
    items = []
    for shape in _shapes(case):
        k, cols = shape[3], shape[0] * shape[1] * shape[2]
        w = _tensor(gen, shape, math.sqrt(2.0 / cols))
        rank = max(1, min(k, cols) // 8)                                                     # gradients: a few directions, and noise
        u, v = torch.empty(k, rank, device="cuda").normal_(0, 1, generator=gen), torch.empty(rank, cols, device="cuda").normal_(0, 1, generator=gen)
        u *= torch.logspace(0, -1.5, rank, device="cuda")
        grad = (u @ v) * (1e-2 / math.sqrt(rank)) + torch.empty(k, cols, device="cuda").normal_(0, 2e-3, generator=gen)
        grad = grad.view(tuple(reversed(shape))).permute(3, 2, 1, 0)
        items.append((w, {"s1": _tensor(gen, shape, 1e-2), "t": 3}, grad, _DECAY, _RATE))
    return dict(case, items=items)


# ------------------------------------------------------------------------------------------------------- plain form
def _logits_lse(x, f, b, labels):
    """log(sum(exp(x f' + b))) per row, 0 for rows without a class."""
    out = torch.empty(x.shape[0], device=x.device)
    for at in range(0, x.shape[0], 2048):
        z = x[at:at + 2048] @ f.t() + b
        top = z.amax(1)
        out[at:at + 2048] = top + (z - top[:, None]).exp().sum(1).log()
    return torch.where(labels > 0, out, torch.zeros_like(out))


def _layernorm(s):
    x = s["x"]
    c = x.shape[2]
    g, b = s["g"].reshape(1, 1, c, 1), s["bias"].reshape(1, 1, c, 1)
    dev = x - x.mean(2, keepdim=True)
    r = 1.0 / ((dev * dev).mean(2, keepdim=True) + _EPSILON).sqrt()
    xh = dev * r
    if not s["back"]:
        return g * xh + b
    dy = s["dzdy"]
    gd = g * dy
    dx = r * (gd - gd.mean(2, keepdim=True) - xh * (gd * xh).mean(2, keepdim=True))
    return dx, (dy * xh).sum((0, 1, 3)).reshape(c, 1), dy.sum((0, 1, 3)).reshape(c, 1)


def _fcloss(s):
    x, f, b, labels = _rows(s["x"]), _rows(s["f"]), s["bias"].reshape(-1), s["labels"]
    n = x.shape[0]
    real, at = labels > 0, (labels.long() - 1).clamp(min=0)
    z = x @ f.t() + b
    if not s["back"]:
        top = z.amax(1)
        lse = top + (z - top[:, None]).exp().sum(1).log()
        lse = torch.where(real, lse, torch.zeros_like(lse))
        terms = torch.where(real, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
        return (terms.sum() / n).reshape(1), lse
    z = (z - s["lse"][:, None]).exp()
    z[torch.arange(n, device=z.device), at] -= 1.0
    z = torch.where(real[:, None], z, torch.zeros((), device=z.device)) / n
    shape = lambda t: t.t().reshape(1, 1, t.shape[1], t.shape[0])                             # noqa: E731
    return shape(z @ f), shape(z.t() @ x), z.sum(0).reshape(-1, 1)


def _muon(s):
    o, out = _MUON, []
    for w, state, grad, decay, rate in s["items"]:
        g = _GRAD_MULT * grad + decay * w
        state["s1"].mul_(o["momentum"]).add_(g)
        u = g + o["momentum"] * state["s1"]
        x = _rows(u)
        rows, cols = x.shape
        x = x / ((x * x).sum(dtype=torch.float64).sqrt().float() + o["epsilon"])
        x = x.t() if rows > cols else x
        for _ in range(o["steps"]):
            p = x @ x.t()
            x = o["a"] * x + (o["b"] * p + o["c"] * (p @ p)) @ x
        x = (x.t() if rows > cols else x).reshape(tuple(reversed(w.shape))).permute(3, 2, 1, 0)
        w.sub_(rate * math.sqrt(max(1.0, rows / cols)) * x)
        out += [w, state["s1"]]
    return out


def run(state):
    op = state["op"]
    if own:
        from matconvnet_b200 import nn
        if op == "layernorm":
            if state["back"]:
                return nn.vl_nnlayernorm(state["x"], state["g"], state["bias"], state["dzdy"], epsilon=_EPSILON)
            return nn.vl_nnlayernorm(state["x"], state["g"], state["bias"], epsilon=_EPSILON)
        if op == "fcloss":
            if state["back"]:
                return nn.vl_nnfcsoftmaxloss(state["x"], state["f"], state["bias"], state["labels"], 1.0, lse=state["lse"])
            return nn.vl_nnfcsoftmaxloss(state["x"], state["f"], state["bias"], state["labels"])
        nn.solver_update_many_("muon", state["items"], _GRAD_MULT, _MUON)
        return [t for w, kept, _, _, _ in state["items"] for t in (w, kept["s1"])]
    return {"layernorm": _layernorm, "fcloss": _fcloss, "muon": _muon}[op](state)


# ------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        x, g, b = (s[k].double() for k in ("x", "g", "bias"))
        c = x.shape[2]
        x = x.movedim(2, -1)
        g, b = g.reshape(-1), b.reshape(-1)
        var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
        r = torch.rsqrt(var + _EPSILON)
        if not case["back"]:
            return ((x - mean) * r * g + b).movedim(-1, 2)
        dy = s["dzdy"].double().movedim(2, -1)
        xh, gd = (x - mean) * r, dy * g
        dx = (gd - gd.sum(-1, keepdim=True) / c - xh * ((gd * xh).sum(-1, keepdim=True) / c)) * r
        return dx.movedim(-1, 2), torch.einsum("hwnc,hwnc->c", dy, xh)[:, None], torch.einsum("hwnc->c", dy)[:, None]
    if case["op"] == "fcloss":
        n, d, k = case["n"], case["d"], case["k"]
        x, f, b = _rows(s["x"]).double(), _rows(s["f"]).double(), s["bias"].double().reshape(-1)
        labels = s["labels"].long()
        dx, df, db = torch.zeros_like(x), torch.zeros_like(f), torch.zeros_like(b)
        lse, loss = torch.zeros(n, device="cuda", dtype=torch.float64), 0.0
        for at in range(0, n, 2048):
            part = slice(at, min(n, at + 2048))
            real = labels[part] > 0
            logp = torch.addmm(b, x[part], f.t())
            if not case["back"]:
                lse[part] = torch.logsumexp(logp, 1) * real
                logp = logp - torch.logsumexp(logp, 1, keepdim=True)
                loss = loss - (torch.gather(logp, 1, (labels[part] - 1).clamp(min=0)[:, None])[:, 0] * real).sum() / n
                continue
            dz = torch.softmax(logp, 1)
            del logp
            dz.scatter_add_(1, (labels[part] - 1).clamp(min=0)[:, None], -torch.ones(dz.shape[0], 1, device="cuda", dtype=torch.float64))
            dz *= real[:, None] / n
            dx[part] = dz @ f
            df.addmm_(dz.t(), x[part])
            db += dz.sum(0)
        if not case["back"]:
            return loss.reshape(1), lse
        return dx.t().reshape(1, 1, d, n), df.t().reshape(1, 1, d, k), db.reshape(k, 1)
    o, out = _MUON, []
    for w, state, grad, decay, rate in s["items"]:
        w, m, grad = (_rows(t).double() for t in (w, state["s1"], grad))
        g = grad * _GRAD_MULT + w * decay
        m = m * o["momentum"] + g
        x = m * o["momentum"] + g
        rows, cols = x.shape
        x = x / (torch.linalg.norm(x) + o["epsilon"])
        gram = (lambda y: x.t() @ y) if rows > cols else (lambda y: y @ x.t())
        for _ in range(o["steps"]):
            p = gram(x)
            y = x @ p if rows > cols else p @ x
            x = o["a"] * x + o["b"] * y + o["c"] * (y @ p if rows > cols else p @ y)
        w = w - (rate * math.sqrt(max(1.0, rows / cols))) * x
        like = state["s1"]
        out += [t.reshape(tuple(reversed(like.shape))).permute(3, 2, 1, 0) for t in (w, m)]
    return out
