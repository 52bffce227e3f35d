"""Performance cases of the 4-bit microscaled products and of distillation.

Each case is one call that a user's program makes: quantising a tensor to 4-bit floating
point in blocks of 32 with a shared power-of-two scale (``quantize``), a linear layer of two
such operands (``linear``), a training step of one (``train``), the largest logits of a
teacher with the mass of the others (``top``), and a step of the distillation loss with its
gradient (``distill``).  ``listed`` names the cases that are always measured and ``draw`` gives
more of the same ranges; ``prepare`` makes what the program holds before the call, ``run``
makes the call (with ``own`` false, the same operator in plain torch), and ``exact`` evaluates
it in 64 bits.
"""

import math

import torch

own = False

DEVICE = torch.device("cuda", 0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}

# Bounds of the drawn cases: the work of the largest listed one of each kind.
MOST_MACS = 2048 * 4096 * 11008
MOST_VALUES = 11008 * 4096
MOST_LOGITS = 2048 * 128000


def _cases():
    # One token's activations: the quantizer alone in a decoding step.
    yield dict(name="quantize-token", op="quantize", type="bf16", n=1, k=4096)
    # A feed-forward weight as it is loaded.
    yield dict(name="quantize-weight", op="quantize", type="fp32", n=11008, k=4096)
    # A decoding step of one sequence: the weight's bytes are all that counts.
    yield dict(name="linear-token", op="linear", type="bf16", n=1, k=4096, o=11008, bias=False)
    # A decoding step of two dozen sequences.
    yield dict(name="linear-batch", op="linear", type="bf16", n=24, k=11008, o=4096, bias=True)
    # A layer whose sizes fit no tile, in FP32.
    yield dict(name="linear-ragged", op="linear", type="fp32", n=777, k=1500, o=1111, bias=True)
    # A prompt of 2048 tokens through a feed-forward projection.
    yield dict(name="linear-prompt", op="linear", type="bf16", n=2048, k=4096, o=11008, bias=False)
    # A training step of a small FP32 classifier layer.
    yield dict(name="train-small", op="train", type="fp32", n=100, k=784, o=512, bias=True)
    # A training step of a feed-forward down projection.
    yield dict(name="train-large", op="train", type="bf16", n=2048, k=11008, o=4096, bias=False)
    # The teacher's top logits for one token of a generation.
    yield dict(name="top-token", op="top", type="fp32", n=1, v=50001, k=20, temperature=1.0)
    # The same for a training batch of 2048 tokens.
    yield dict(name="top-batch", op="top", type="bf16", n=2048, v=128000, k=64, temperature=2.0)
    # An image classifier's batch, some entries and rows left out.
    yield dict(name="distill-classes", op="distill", type="fp32", n=32, v=1000, k=10,
               temperature=4.0, tail=True, ragged=True, weights=True)
    # A language model's batch of 2048 tokens.
    yield dict(name="distill-tokens", op="distill", type="bf16", n=2048, v=128000, k=64,
               temperature=1.0, tail=True, ragged=False, weights=False)


def listed():
    return list(_cases())


def _spread(rng, low, high):
    """A whole number between low and high, evenly over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "train", "top", "distill"))
    kind = rng.choice(tuple(TYPES))
    while True:
        if op == "quantize":
            n, k = _spread(rng, 1, 11008), _spread(rng, 32, 11008)
            if n * k <= MOST_VALUES:
                return dict(op=op, type=kind, n=n, k=k)
        elif op in ("linear", "train"):
            n, k, o = _spread(rng, 1, 4096), _spread(rng, 64, 11008), _spread(rng, 10, 11008)
            if n * k * o <= MOST_MACS // (4 if kind == "fp32" else 1):
                return dict(op=op, type=kind, n=n, k=k, o=o, bias=rng.random() < 0.5)
        else:
            n, v, k = _spread(rng, 1, 4096), _spread(rng, 1000, 131072), _spread(rng, 1, 256)
            if n * v <= MOST_LOGITS // (2 if kind == "fp32" else 1):
                case = dict(op=op, type=kind, n=n, v=v, k=k,
                            temperature=rng.choice((0.5, 1.0, 2.0, 4.0)))
                if op == "distill":
                    case.update(tail=rng.random() < 0.7, ragged=rng.random() < 0.3,
                                weights=rng.random() < 0.3)
                return case


# ---------------------------------------------------------------------------
# 4-bit blocks in plain torch
# ---------------------------------------------------------------------------
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantized(x):
    """(FP32 elements, FP32 scales) of x [n, k] in blocks of 32: [n, b, 32] and [n, b, 1]."""
    n, k = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -k % 32)).reshape(n, -1, 32)
    exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True)).exponent - 3
    scale = torch.ldexp(torch.ones_like(exponent, dtype=torch.float32),
                        exponent.clamp(min=-126))
    y = blocks / scale
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = torch.round(size / step).mul(step).clamp(max=6.0)
    return torch.copysign(size, y), scale


def _rounded(x):
    """The FP32 values that x's 4-bit codes stand for."""
    element, scale = _quantized(x)
    return (element * scale).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _packed(x):
    """Codes uint8 [n, 128 b] (low half first) and scale bytes uint8 [n, 8 b] of x [n, k],
    b = ceil(k / 256): rows of whole 256-value segments, zeros past k."""
    n, k = x.shape
    element, scale = _quantized(torch.nn.functional.pad(x, (0, -k % 256)))
    grid = torch.tensor(MAGNITUDES, device=x.device)
    code = torch.bucketize(element.abs(), grid) + 8 * torch.signbit(element)
    code = code.reshape(n, -1, 2).to(torch.uint8)
    byte = torch.frexp(scale).exponent + 126
    return code[..., 0] | code[..., 1] << 4, byte.reshape(n, -1).to(torch.uint8)


def _unpacked(codes, scales, k, dtype):
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=dtype,
                         device=codes.device)
    values = table[torch.stack((codes & 15, codes >> 4), -1).long()].reshape(len(codes), -1, 32)
    scale = torch.ldexp(torch.ones(scales.shape, dtype=dtype, device=codes.device),
                        scales.int() - 127)
    return (values * scale[..., None]).reshape(len(codes), -1)[:, :k]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _activations(gen, n, k):
    """Unit normals with every hundredth channel 20 times larger."""
    x = torch.randn(n, k, generator=gen, device=DEVICE)
    x[:, torch.randperm(k, generator=gen, device=DEVICE)[:max(1, k // 100)]] *= 20
    return x


def _logits(gen, n, v):
    """Logits of a peaked distribution: most values low, a few of each row far above."""
    s = torch.randn(n, v, generator=gen, device=DEVICE)
    return s.clamp(min=0).pow_(3).mul_(0.15).add_(s, alpha=2.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, n = TYPES[case["type"]], case["n"]
    state = dict(case=case)
    if case["op"] == "quantize":
        state["x"] = _activations(gen, n, case["k"]).to(dtype)
    elif case["op"] in ("linear", "train"):
        k, o, train = case["k"], case["o"], case["op"] == "train"
        state["x"] = _activations(gen, n, k).to(dtype).requires_grad_(train)
        weight = 0.02 * torch.randn(o, k, generator=gen, device=DEVICE)
        if train:
            state["weight"] = weight.to(dtype).requires_grad_(True)
            state["dy"] = (0.01 * torch.randn(n, o, generator=gen, device=DEVICE)).to(dtype)
        else:   # a layer's weight is kept in its 4-bit form
            state["codes"], state["scales"] = _packed(weight)
        state["bias"] = None
        if case["bias"]:
            bias = 0.1 * torch.randn(o, generator=gen, device=DEVICE)
            state["bias"] = bias.to(dtype).requires_grad_(train)
    else:
        v, k = case["v"], min(case["k"], case["v"])
        state["logits"] = _logits(gen, n, v).to(dtype)
        if case["op"] == "distill":
            state["logits"].requires_grad_(True)
            # A teacher that agrees with the student up to noise.
            teacher = state["logits"].detach().float()
            teacher = teacher + torch.randn(n, v, generator=gen, device=DEVICE)
            values, indices, tail = _top(teacher.to(dtype), k, case["temperature"])
            if case["ragged"]:
                lost = torch.rand(n, k, generator=gen, device=DEVICE) < 0.2
                lost[:, 0] = False
                indices = indices.masked_fill(lost, -1)
            state["values"], state["indices"] = values, indices
            state["tail"] = tail if case["tail"] else None
            state["row_weight"] = None
            if case["weights"]:
                kept = torch.rand(n, generator=gen, device=DEVICE) < 0.8
                kept[0] = True
                state["row_weight"] = kept.float()
    return state


# ---------------------------------------------------------------------------
# The operators in plain torch, in 32 bits
# ---------------------------------------------------------------------------
def _log_sum(z):
    """log(sum(exp(z))) over the last dimension; -inf where nothing is left."""
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    return (top + torch.exp(z - top).sum(-1, keepdim=True).log()).squeeze(-1)


def _top(logits, k, temperature):
    """The k largest of each row in order, the lowest index first among equals, and
    log(sum(exp(logits / T))) of the others."""
    bits = (logits.float() + 0.0).view(torch.int32)   # -0 as 0
    order = bits ^ (bits >> 31 & 0x7FFFFFFF)     # whole numbers in the order of the values
    key = (order.long() << 32) + (2**31 - torch.arange(logits.shape[1], device=logits.device))
    indices = torch.topk(key, k, dim=1).indices
    z = logits.float() / temperature
    tail = _log_sum(z.scatter(1, indices, -math.inf))
    return logits.gather(1, indices), indices, tail


def _plain_distill(state):
    case, t = state["case"], state["case"]["temperature"]
    logits, indices, n = state["logits"].detach(), state["indices"], state["case"]["n"]
    z = logits.float() / t
    kept = indices >= 0
    at = indices.clamp(min=0)
    teacher = torch.where(kept, state["values"].float() / t, -math.inf)
    tail = state["tail"] if case["tail"] else torch.full((n,), -math.inf, device=DEVICE)
    teacher = torch.cat((teacher, tail[:, None]), 1)
    log_p = teacher - _log_sum(teacher)[:, None]
    p = log_p.exp()
    marked = torch.zeros(n, z.shape[1] + 1, dtype=torch.bool, device=DEVICE)
    marked = marked.scatter_(1, torch.where(kept, indices, z.shape[1]), True)[:, :-1]
    rest = z.masked_fill(marked, -math.inf)
    total, others = _log_sum(z), _log_sum(rest)
    entries = torch.where(kept, z.gather(1, at), -math.inf)
    log_q = torch.cat((entries, others[:, None]), 1) - total[:, None]
    # p log(p/q) - p + q of every bucket: the same sum, as p and q both add up to 1, but of terms
    # that are never negative and so do not cancel where p is near q.
    d = torch.where(p > 0, log_p - log_q, 0.0)
    near = d * d * (0.5 - d * (1 / 6 - d * (1 / 24 - d * (1 / 120 - d / 720))))
    term = p * torch.where(d.abs() < 0.25, near, d + torch.expm1(-d))
    loss = torch.where(p > 0, term, log_q.exp()).sum(1) * t * t
    weight = state["row_weight"]
    weight = torch.ones(n, device=DEVICE) if weight is None else weight
    share = weight / weight.sum()
    grad = torch.exp(z - total[:, None]) - p[:, -1:] * torch.exp(rest - others[:, None])
    grad = grad.scatter_add(1, at, torch.where(kept, -p[:, :-1], 0.0))
    return dict(loss=(share * loss).sum(), dlogits=(grad * (t * share[:, None])).to(logits.dtype))


def _plain(state):
    case = state["case"]
    dtype = TYPES[case["type"]]
    if case["op"] == "quantize":
        return _rounded(state["x"]).to(dtype)
    if case["op"] == "linear":
        y = _rounded(state["x"]) @ _unpacked(state["codes"], state["scales"], case["k"],
                                             torch.float32).T
        return (y if state["bias"] is None else y + state["bias"].float()).to(dtype)
    if case["op"] == "train":
        x, weight = _rounded(state["x"].detach()), _rounded(state["weight"].detach())
        dy = state["dy"].float()
        y = x @ weight.T
        out = dict(dx=(dy @ weight).to(dtype), dw=(dy.T @ x).to(dtype))
        if state["bias"] is not None:
            y = y + state["bias"].detach().float()
            out["db"] = dy.sum(0).to(dtype)
        return dict(out, y=y.to(dtype))
    if case["op"] == "top":
        return dict(zip(("values", "indices", "tail"),
                        _top(state["logits"], min(case["k"], case["v"]), case["temperature"])))
    return _plain_distill(state)


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _framework(state):
    import memfast_amd as memfast

    case = state["case"]
    if case["op"] == "quantize":
        return memfast.mx_quantize(state["x"]).dequantize(TYPES[case["type"]])
    if case["op"] == "linear":
        weight = memfast.MXTensor(state["codes"], state["scales"], (case["o"], case["k"]))
        return memfast.mx_linear(state["x"], weight, state["bias"])
    if case["op"] == "train":
        inputs = [state["x"], state["weight"]]
        if state["bias"] is not None:
            inputs.append(state["bias"])
        y = memfast.mx_linear(state["x"], state["weight"], state["bias"])
        grads = torch.autograd.grad(y, inputs, state["dy"])
        return dict(zip(("dx", "dw", "db"), grads), y=y.detach())
    if case["op"] == "top":
        top = memfast.top_logits(state["logits"], min(case["k"], case["v"]),
                                 temperature=case["temperature"])
        return dict(zip(("values", "indices", "tail"), top))
    loss = memfast.distillation_loss(state["logits"], state["values"], state["indices"],
                                     state["tail"], temperature=case["temperature"],
                                     weight=state["row_weight"])
    return dict(loss=loss.detach(), dlogits=torch.autograd.grad(loss, state["logits"])[0])


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b, n = BYTES[case["type"]], case["n"]
    if case["op"] == "quantize":
        k = case["k"]
        return dict(bytes=n * k * (2 * b + 17 / 32), flops=0)
    if case["op"] in ("linear", "train"):
        k, o = case["k"], case["o"]
        bias = b * o if case["bias"] else 0
        if case["op"] == "linear":
            return dict(bytes=b * n * (k + o) + o * k * 17 / 32 + bias, flops=2 * n * k * o)
        # x, w, dy in; y, dx, dw out (and the bias and its gradient).
        return dict(bytes=2 * b * (n * k + o * k + n * o) + 2 * bias, flops=6 * n * k * o)
    v, k = case["v"], min(case["k"], case["v"])
    if case["op"] == "top":
        return dict(bytes=n * (v * b + k * (b + 8) + 4), flops=0)
    return dict(bytes=n * (2 * v * b + k * (b + 8) + 8), flops=0)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rounded(x):
    """The nearest multiple of the block's scale among the magnitudes; a value halfway between
    two takes the one whose last bit is 0."""
    n, k = x.shape
    y = torch.zeros(n, (k + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    y[:, :k] = x.detach().double()
    y = y.view(n, -1, 32)
    peak = y.abs().max(-1, keepdim=True).values
    scale = torch.pow(2.0, (torch.floor(torch.log2(peak)) - 2).clamp(min=-126))
    size = y.abs() / scale
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    index = torch.bucketize(size, middle)
    for odd in (0.75, 1.75, 3.5):
        index += size == odd
    return (torch.sign(y) * grid[index] * scale).view(n, -1)[:, :k]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_rounded(state["x"])
    if case["op"] == "linear":
        weight = _unpacked(state["codes"], state["scales"], case["k"], torch.float64)
        y = torch.matmul(_exact_rounded(state["x"]), weight.T.contiguous())
        return y if state["bias"] is None else y + state["bias"].double()
    if case["op"] == "train":
        x, weight = _exact_rounded(state["x"]), _exact_rounded(state["weight"])
        dy = state["dy"].double()
        y = torch.matmul(x, weight.T.contiguous())
        out = dict(dx=torch.matmul(dy, weight), dw=torch.matmul(dy.T.contiguous(), x))
        if state["bias"] is not None:
            y = y + state["bias"].detach().double()
            out["db"] = dy.sum(0)
        return dict(out, y=y)
    t = case["temperature"]
    z = state["logits"].detach().double() / t
    if case["op"] == "top":
        k = min(case["k"], case["v"])
        ordered, indices = torch.sort(state["logits"].double(), dim=1, descending=True,
                                      stable=True)
        return dict(values=ordered[:, :k], indices=indices[:, :k],
                    tail=torch.logsumexp(ordered[:, k:] / t, 1))
    z.requires_grad_(True)
    q = torch.log_softmax(z, 1)
    kept = state["indices"] >= 0
    values = (state["values"].double() / t).masked_fill(~kept, -math.inf)
    if case["tail"]:
        values = torch.cat((values, state["tail"].double()[:, None]), 1)
    log_p = torch.log_softmax(values, 1)
    at = state["indices"].clamp(min=0)
    log_q = q.gather(1, at)
    if case["tail"]:
        inside = torch.zeros_like(z, dtype=torch.int32).scatter_add_(1, at, kept.int()) > 0
        log_q = torch.cat((log_q, torch.logsumexp(q.masked_fill(inside, -math.inf), 1)[:, None]), 1)
    terms = torch.where(log_p > -math.inf, log_p.exp() * (log_p.clamp(min=-1e300) - log_q), 0.0)
    weight = state["row_weight"]
    share = torch.full_like(terms[:, 0], 1 / case["n"]) if weight is None else \
        weight.double() / weight.double().sum()
    loss = (share * terms.sum(1)).sum() * t * t
    return dict(loss=loss.detach(), dlogits=torch.autograd.grad(loss, z)[0] / t)
