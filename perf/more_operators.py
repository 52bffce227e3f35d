"""Performance cases of gated linear recurrences, of dropout and of products with 4-bit weights.

A recurrent model without hidden projections takes all its projections of a sequence at once and
leaves a gated linear recurrence per channel.  The cases are what such a model's program calls: one
step of it for a batch of streams (``step``), a whole sequence (``scan``), a sequence with its gradients
(``learn``), the dropout between layers with its gradient (``dropout``), and the projections of a
served model, held as 4-bit integers with a scale for each group of inputs (``held``).

``listed`` names the cases that are always measured and ``draw`` gives more of the same ranges;
``prepare`` makes what the program holds before the call, ``run`` makes the call (with ``own`` false,
the same operator in plain torch), and ``exact`` evaluates it in 64 bits.
"""

import math

import numpy
import torch

own = False

DEVICE = torch.device("cuda", 0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}

# Bounds of the drawn cases: the work of the largest listed one of each kind.
MOST_STATES = 8 * 4096 * 2048
MOST_VALUES = 8192 * 4096
MOST_MACS = 2048 * 4096 * 11008


def _cases():
    # One token of 32 streams that a server advances together.
    yield dict(name="step-streams", op="step", type="bf16", steps=1, batch=32, width=1024,
               tanh=True, state=True, lengths=False, reverse=False, batch_first=False)
    # A padded batch of sequences through the backward direction, with sizes that fit nothing.
    yield dict(name="scan-ragged", op="scan", type="fp32", steps=777, batch=5, width=333,
               tanh=True, state=True, lengths=True, reverse=True, batch_first=True)
    # One long document: few channels and very many steps.
    yield dict(name="scan-document", op="scan", type="bf16", steps=65536, batch=1, width=512,
               tanh=False, state=False, lengths=False, reverse=False, batch_first=False)
    # A training step of a small FP32 layer over a padded batch.
    yield dict(name="learn-small", op="learn", type="fp32", steps=100, batch=16, width=128,
               tanh=True, state=False, lengths=True, reverse=False, batch_first=True)
    # A training step of a wide layer over 8 sequences of 4096 tokens.
    yield dict(name="learn-large", op="learn", type="bf16", steps=4096, batch=8, width=2048,
               tanh=True, state=True, lengths=False, reverse=False, batch_first=True)
    # Dropout between two layers of a small network.
    yield dict(name="dropout-small", op="dropout", type="fp32", rows=100, width=512, p=0.5,
               residual=False)
    # Dropout of 8192 tokens' outputs that join the residual stream.
    yield dict(name="dropout-residual", op="dropout", type="bf16", rows=8192, width=4096, p=0.1,
               residual=True)
    # A decoding step of one sequence: the weight's bytes are all that counts.
    yield dict(name="held-token", op="held", type="bf16", n=1, k=4096, o=11008, group=32,
               zeros=False, bias=False)
    # A decoding step of two dozen sequences with weights imported with zero points.
    yield dict(name="held-batch", op="held", type="fp16", n=24, k=11008, o=4096, group=128,
               zeros=True, bias=True)
    # An FP32 layer whose sizes fit no tile.
    yield dict(name="held-ragged", op="held", type="fp32", n=77, k=1500, o=1111, group=64,
               zeros=False, bias=True)
    # A prompt of 2048 tokens through the same projection.
    yield dict(name="held-prompt", op="held", type="bf16", n=2048, k=4096, o=11008, group=128,
               zeros=False, bias=False)


def listed():
    return list(_cases())


def _spread(rng, low, high):
    """A whole number between low and high, evenly over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("step", "scan", "learn", "dropout", "held"))
    kind = rng.choice(tuple(TYPES))
    share = 2 if kind == "fp32" else 1
    while True:
        if op == "dropout":
            rows, width = _spread(rng, 1, 8192), _spread(rng, 8, 8192)
            if rows * width <= MOST_VALUES // share:
                return dict(op=op, type=kind, rows=rows, width=width,
                            p=rng.choice((0.05, 0.1, 0.2, 0.5)), residual=rng.random() < 0.5)
        elif op == "held":
            n, k, o = _spread(rng, 1, 2048), _spread(rng, 64, 11008), _spread(rng, 10, 11008)
            if n * k * o <= MOST_MACS // (2 * share):
                return dict(op=op, type=kind, n=n, k=k, o=o, group=rng.choice((32, 64, 128)),
                            zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
        else:
            steps = 1 if op == "step" else _spread(rng, 2, 65536 if op == "scan" else 8192)
            batch, width = _spread(rng, 1, 64), _spread(rng, 16, 4096)
            if steps * batch * width <= MOST_STATES // share:
                return dict(op=op, type=kind, steps=steps, batch=batch, width=width,
                            tanh=rng.random() < 0.5, state=op == "step" or rng.random() < 0.5,
                            lengths=op != "step" and rng.random() < 0.4,
                            reverse=op != "step" and rng.random() < 0.4,
                            batch_first=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _packed(q):
    """Codes uint8 [ceil(o / 16), ceil(k / 128), 1024] of whole numbers q [o, k] in 0 .. 15: tiles of
    16 outputs by 128 inputs.  A tile's bytes run over (input / 8) % 4, the output, input / 32 and
    input % 4; a byte holds input % 8 < 4 in its lower half and the input 4 further in its upper."""
    o, k = q.shape
    q = torch.nn.functional.pad(q, (0, -k % 128, 0, -o % 16))
    tiles = q.view(-(-o // 16), 16, -(-k // 128), 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)
    return (tiles[..., 0] | tiles[..., 1] << 4).reshape(-(-o // 16), -(-k // 128), 1024)


def _by_tile(table):
    """[ceil(o / 16), groups, 16] of a table [o, groups], with zeros past o."""
    o, groups = table.shape
    table = torch.nn.functional.pad(table, (0, 0, 0, -o % 16))
    return table.view(-1, 16, groups).transpose(1, 2).contiguous()


def _held(gen, case, dtype):
    """A trained weight's codes, scales and zero points."""
    k, o, group = case["k"], case["o"], case["group"]
    groups = -(-k // group)
    weight = 0.02 * _normal(gen, o, k)
    spans = torch.nn.functional.pad(weight, (0, -k % group)).view(o, groups, group)
    low, high = spans.amin(-1), spans.amax(-1)
    if case["zeros"]:
        scales = ((high - low) / 15).to(dtype)
        zeros = torch.round(-low / scales.float()).clamp(0, 15)
    else:
        scales = (torch.maximum(-low, high) / 7).to(dtype)
        zeros = torch.full_like(low, 8.0)
    q = torch.round(spans / scales.float()[..., None] + zeros[..., None]).clamp(0, 15)
    q = q.view(o, -1)[:, :k].to(torch.uint8)
    return _packed(q), _by_tile(scales), _by_tile(zeros.to(torch.uint8)) if case["zeros"] else None


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = dict(case=case)
    if case["op"] == "dropout":
        shape = case["rows"], case["width"]
        state["x"] = _normal(gen, *shape).to(dtype).requires_grad_(True)
        state["residual"] = _normal(gen, *shape).to(dtype).requires_grad_(True) \
            if case["residual"] else None
        state["dy"] = (0.01 * _normal(gen, *shape)).to(dtype)
        state["seed"], state["event"] = 1000003 * seed + 12345, seed % 1000
    elif case["op"] == "held":
        state["codes"], state["scales"], state["zeros"] = _held(gen, case, dtype)
        state["x"] = _normal(gen, case["n"], case["k"]).to(dtype)
        state["bias"] = (0.1 * _normal(gen, case["o"])).to(dtype) if case["bias"] else None
    else:
        steps, batch, width = case["steps"], case["batch"], case["width"]
        train = case["op"] == "learn"
        lead = (batch, steps) if case["batch_first"] else (steps, batch)
        # Channels that forget within a few steps and others that remember hundreds.
        projected = _normal(gen, *lead, 2 * width)
        projected[..., :width] += 1.5 + 1.5 * _normal(gen, width)
        state["projected"] = projected.to(dtype).requires_grad_(train)
        state["state"] = _normal(gen, batch, width).clamp(-1, 1).requires_grad_(train) \
            if case["state"] else None
        state["lengths"] = None
        if case["lengths"]:
            state["lengths"] = torch.randint(0, steps + 1, (batch,), generator=gen, device=DEVICE)
            state["lengths"][0] = steps
        if train:
            state["doutput"] = (0.01 * _normal(gen, *lead, width)).to(dtype)
            state["dfinal"] = 0.01 * _normal(gen, batch, width)
    return state


# ---------------------------------------------------------------------------
# The operators in plain torch
# ---------------------------------------------------------------------------
def _scan(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along the first dimension, by doubling."""
    distance = 1
    while distance < len(b):
        b = torch.cat((b[:distance], torch.addcmul(b[distance:], a[distance:], b[:-distance])))
        a = torch.cat((a[:distance], a[distance:] * a[:-distance]))
        distance *= 2
    return b


def _time_first(x, case):
    """x with its steps first and in the order in which they are taken."""
    x = x.transpose(0, 1) if case["batch_first"] else x
    return x.flip(0) if case["reverse"] else x


def _as_given(x, case):
    x = x.flip(0) if case["reverse"] else x
    return x.transpose(0, 1) if case["batch_first"] else x


def _plain_recurrence(state):
    case = state["case"]
    dtype, width = TYPES[case["type"]], case["width"]
    x = _time_first(state["projected"].detach().float(), case)
    gate, value = x[..., :width], x[..., width:]
    start = torch.zeros_like(value[0]) if state["state"] is None else state["state"].detach()
    keep, take = torch.sigmoid(gate), torch.sigmoid(-gate)
    if case["tanh"]:
        value = torch.tanh(value)
    added = take * value
    live = None
    if state["lengths"] is not None:
        live = torch.arange(case["steps"], device=DEVICE)[:, None] < state["lengths"]
        live = (live.flip(0) if case["reverse"] else live)[..., None]
        keep, added = torch.where(live, keep, 1.0), torch.where(live, added, 0.0)
    first = torch.addcmul(added[:1], keep[:1], start[None])
    h = _scan(keep, torch.cat((first, added[1:])))
    output = h if live is None else torch.where(live, h, 0.0)
    out = dict(output=_as_given(output, case).to(dtype).contiguous(), final=h[-1].clone())
    if case["op"] != "learn":
        return out
    g = _time_first(state["doutput"].float(), case)
    g = g if live is None else torch.where(live, g, 0.0)
    g = torch.cat((g[:-1], g[-1:] + state["dfinal"][None]))
    later = torch.cat((keep[1:], torch.ones_like(keep[:1])))
    g = _scan(later.flip(0), g.flip(0)).flip(0)
    before = torch.cat((start[None], h[:-1]))
    dgate = g * (before - value) * keep * take
    dvalue = g * take
    if case["tanh"]:
        dvalue = dvalue * (1 - value * value)
    dx = torch.cat((dgate, dvalue), -1)
    dx = dx if live is None else torch.where(live, dx, 0.0)
    out["dprojected"] = _as_given(dx, case).to(dtype).contiguous()
    if state["state"] is not None:
        out["dstate"] = keep[0] * g[0]
    return out


def _philox(words, key):
    """Ten rounds of Philox 4x32 (Salmon et al. 2011) on four int64 tensors of 32-bit words."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = words
    k0, k1 = key & low, key >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57      # the lower 64 bits, whatever their sign
        c0, c1, c2, c3 = p1 >> 32 & low ^ c1 ^ k0, p1 & low, p0 >> 32 & low ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return c0, c1, c2, c3


def _share(p):
    """Of 65536 equally likely numbers, how many drop a value."""
    return round(p * 65536)


def _plain_dropout(state):
    case, x = state["case"], state["x"].detach()
    dropped = _share(case["p"])
    block = torch.arange(-(-x.numel() // 8), device=DEVICE)
    event = torch.full_like(block, state["event"])
    words = _philox((block & 0xFFFFFFFF, block >> 32, event & 0xFFFFFFFF, event >> 32),
                    state["seed"])
    words = torch.stack(words, -1)
    numbers = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:x.numel()]
    factor = torch.where(numbers >= dropped, 65536 / (65536 - dropped), 0.0).view_as(x)
    y = x.float() * factor
    if state["residual"] is not None:
        y = y + state["residual"].detach().float()
    out = dict(y=y.to(x.dtype), dx=(state["dy"].float() * factor).to(x.dtype))
    if state["residual"] is not None:
        out["dresidual"] = state["dy"]
    return out


def _plain_held(state):
    case = state["case"]
    k, o, group = case["k"], case["o"], case["group"]
    codes = state["codes"]
    q = torch.stack((codes & 15, codes >> 4), -1).view(*codes.shape[:2], 4, 16, 4, 4, 2)
    q = q.permute(0, 3, 1, 4, 2, 6, 5).reshape(16 * codes.shape[0], -1)[:o, :k].float()

    def spread(table):
        table = table.float().transpose(1, 2).reshape(-1, table.shape[1])[:o]
        return table.repeat_interleave(group, 1)[:, :k]

    zeros = 8.0 if state["zeros"] is None else spread(state["zeros"])
    y = state["x"].float() @ (spread(state["scales"]) * (q - zeros)).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _framework(state):
    import memfast_amd as memfast

    case = state["case"]
    if case["op"] == "dropout":
        x, residual = state["x"], state["residual"]
        y = memfast.dropout(x, case["p"], seed=state["seed"], event=state["event"],
                            residual=residual)
        inputs = (x,) if residual is None else (x, residual)
        grads = torch.autograd.grad(y, inputs, state["dy"])
        return dict(zip(("dx", "dresidual"), grads), y=y.detach())
    if case["op"] == "held":
        weight = memfast.Int4Tensor(state["codes"], state["scales"], (case["o"], case["k"]),
                                    group=case["group"], zeros=state["zeros"])
        return memfast.int4_linear(state["x"], weight, state["bias"])
    output, final = memfast.gated_recurrence(
        state["projected"], state["state"], activation="tanh" if case["tanh"] else None,
        lengths=state["lengths"], reverse=case["reverse"], batch_first=case["batch_first"])
    if case["op"] != "learn":
        return dict(output=output, final=final)
    names, inputs = ["dprojected"], [state["projected"]]
    if state["state"] is not None:
        names.append("dstate")
        inputs.append(state["state"])
    grads = torch.autograd.grad((output, final), inputs, (state["doutput"], state["dfinal"]))
    return dict(zip(names, grads), output=output.detach(), final=final.detach())


def run(state):
    if own:
        return _framework(state)
    op = state["case"]["op"]
    return (_plain_dropout if op == "dropout" else _plain_held if op == "held" else
            _plain_recurrence)(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "dropout":
        # x and dy in, y and dx out; the residual in (its gradient is dy itself).
        return dict(bytes=(5 if case["residual"] else 4) * b * case["rows"] * case["width"], flops=0)
    if case["op"] == "held":
        n, k, o = case["n"], case["k"], case["o"]
        groups = -(-k // case["group"])
        table = (b + (1 if case["zeros"] else 0)) * o * groups + (b * o if case["bias"] else 0)
        return dict(bytes=b * n * (k + o) + o * k / 2 + table, flops=2 * n * k * o)
    train, states = case["op"] == "learn", case["batch"] * case["width"]
    n = case["steps"] * states
    # Gates and candidates in, states out; for gradients dy in, those of gates and candidates out.
    held = 4 * states * (2 if case["state"] else 1)
    return dict(bytes=(6 if train else 3) * b * n + held * (2 if train else 1), flops=0)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_recurrence(state):
    case = state["case"]
    train, width = case["op"] == "learn", case["width"]
    x = state["projected"].detach().double()
    x = (x.transpose(0, 1) if case["batch_first"] else x).contiguous().requires_grad_(train)
    start = torch.zeros(x.shape[1], width, dtype=torch.float64, device=DEVICE)
    if state["state"] is not None:
        start = state["state"].detach().double()
    start.requires_grad_(train)
    with torch.set_grad_enabled(train):
        keep = 1 / (1 + torch.exp(-x[..., :width]))
        value = torch.tanh(x[..., width:]) if case["tanh"] else x[..., width:]
        taken = (1 - keep) * value
        h, rows = start, [None] * len(x)
        inside = None
        if state["lengths"] is not None:
            inside = (torch.arange(len(x), device=DEVICE)[:, None] < state["lengths"])[..., None]
            blank = torch.zeros_like(h)
            inside = inside.unbind(0)
        keep, taken = keep.unbind(0), taken.unbind(0)
        for t in reversed(range(len(x))) if case["reverse"] else range(len(x)):
            after = keep[t] * h + taken[t]
            h = after if inside is None else torch.where(inside[t], after, h)
            rows[t] = h if inside is None else torch.where(inside[t], h, blank)
        output = torch.stack(rows, 1 if case["batch_first"] else 0)
    out = dict(output=output.detach(), final=h.detach())
    if train:
        dx, dstart = torch.autograd.grad((output, h), (x, start),
                                         (state["doutput"].double(), state["dfinal"].double()))
        out["dprojected"] = dx.transpose(0, 1) if case["batch_first"] else dx
        if state["state"] is not None:
            out["dstate"] = dstart
    return out


def _exact_numbers(count, seed, event):
    """The 16-bit numbers of Philox 4x32-10 for the counters (block, event), in numpy's uint64."""
    u64 = numpy.uint64
    half, low = u64(32), u64(0xFFFFFFFF)
    block = numpy.arange(-(-count // 8), dtype=u64)
    c = numpy.empty((4, len(block)), dtype=u64)
    c[0], c[1], c[2], c[3] = block & low, block >> half, event & 0xFFFFFFFF, event >> 32
    for turn in range(10):
        k0 = u64((seed + turn * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = u64(((seed >> 32) + turn * 0xBB67AE85) & 0xFFFFFFFF)
        left, right = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c[0], c[2] = (right >> half) ^ c[1] ^ k0, (left >> half) ^ c[3] ^ k1
        c[1], c[3] = right & low, left & low
    return numpy.ascontiguousarray(c.T.astype("<u4")).view("<u2").reshape(-1)[:count]


def _exact_held(state):
    case, codes = state["case"], state["codes"]
    o = torch.arange(case["o"], device=DEVICE)[:, None]
    k = torch.arange(case["k"], device=DEVICE)
    at = (o // 16 * codes.shape[1] + k // 128) * 1024
    at = at + k // 8 % 4 * 256 + o % 16 * 16 + k % 128 // 32 * 4 + k % 4
    q = codes.view(-1)[at] >> (k // 4 % 2 * 4).to(torch.uint8) & 15
    where = o // 16, k // case["group"], o % 16
    zero = 8 if state["zeros"] is None else state["zeros"][where].double()
    weight = state["scales"][where].double() * (q.double() - zero)
    y = torch.matmul(state["x"].double(), weight.T.contiguous())
    return y if state["bias"] is None else y + state["bias"].double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "held":
        return _exact_held(state)
    if case["op"] != "dropout":
        return _exact_recurrence(state)
    x, dropped = state["x"].detach(), _share(case["p"])
    numbers = _exact_numbers(x.numel(), state["seed"], state["event"])
    kept = torch.from_numpy(numbers.astype("int32") >= dropped).to(DEVICE).view_as(x)
    y = torch.where(kept, x.double() / (1 - dropped / 65536), 0.0)
    out = dict(dx=torch.where(kept, state["dy"].double() / (1 - dropped / 65536), 0.0))
    if state["residual"] is not None:
        y, out["dresidual"] = y + state["residual"].detach().double(), state["dy"].double()
    return dict(out, y=y)
