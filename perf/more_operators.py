"""Performance cases of the operators that a label field is trained with and answers with, beside those of operators.py.

A field's training step against given labels scores the labels' log probabilities, carries their gradient back and updates
table, head and whatever else is trained; its answers come from a head held in 4 bits, as log probabilities with the likeliest
alternatives. A case is one pass through one operator:

  adamw      one step over many tensors, moments in 32 bits or in 8 (returned as the values that they stand for, as they are
             read to be saved)
  logprobs   log probabilities of given labels, entropies and top alternatives of rows of logits: alone ("score"), with the
             gradient in one pass ("step"), or with the gradient in a later call from upstream gradients of both ("apart")
  quantize4  rows in microscaled 4-bit blocks of 32, returned as the values that they stand for
  matmul4    product of two matrices in such blocks
  linear4    rows quantised so and multiplied with a weight held so

`run` computes them in elementary float32 torch operations, or with gsx_amd where `own` is true.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
HELD = 128  # values of a block of moments
BLOCK = 32  # values of a 4-bit block
VALUES4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # table and head of the label-field example: what a call costs
        dict(name="adamw_field", kind="adamw", tensors=2, largest=512_000, param="f32", grad="f32", bits=32),
        # tensors of very different, odd sizes, trained in 16 bits
        dict(name="adamw_odd", kind="adamw", tensors=61, largest=300_001, param="bf16", grad="bf16", bits=32),
        # 48 tensors of 102M values in all with 16-bit gradients, moments in 8 bits
        dict(name="adamw_held", kind="adamw", tensors=48, largest=8_388_608, param="f32", grad="bf16", bits=8),
        # the next token of one query over a large vocabulary, with 20 alternatives
        dict(name="logprobs_token", kind="logprobs", rows=1, vocab=131072, top=20, dtype="f32", temperature=1.0,
             mode="score", masked=0.0, blocked=0.01),
        # a label for each pixel of a 640x480 frame: loss and gradient of a training step, and the three likeliest labels
        dict(name="logprobs_pixels", kind="logprobs", rows=307_200, vocab=150, top=3, dtype="bf16", temperature=1.0,
             mode="step", masked=0.1, blocked=0.0),
        # a batch against an odd vocabulary, gradients of log probabilities and entropies in a later call
        dict(name="logprobs_vocab", kind="logprobs", rows=4096, vocab=65537, top=8, dtype="bf16", temperature=2.0,
             mode="apart", masked=0.1, blocked=0.01),
        # a head of odd sizes laid out for answering
        dict(name="quantize4_odd", kind="quantize4", rows=1001, cols=4098, dtype="f32"),
        # a wide square weight
        dict(name="quantize4_large", kind="quantize4", rows=8192, cols=8192, dtype="bf16"),
        # two matrices of odd sizes
        dict(name="matmul4_odd", kind="matmul4", m=2333, n=3001, k=4090, dtype="f32"),
        # the logits of one query: a weight of 71 MB read for a single row
        dict(name="linear4_token", kind="linear4", m=1, n=32768, k=4096, dtype="bf16", out="f32"),
        # a head of 150 labels on the pixels of a 640x480 frame of 128 features
        dict(name="linear4_pixels", kind="linear4", m=307_200, n=150, k=128, dtype="bf16", out="bf16"),
        # a batch of 8192 rows through a wide square layer
        dict(name="linear4_large", kind="linear4", m=8192, n=8192, k=8192, dtype="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("adamw", "logprobs", "quantize4", "matmul4", "linear4"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if kind == "adamw":
        tensors = _log(rng, 1, 200)
        return dict(kind=kind, tensors=tensors, largest=_log(rng, 1, min(33_554_432, 268_435_456 // tensors)), param=dtype,
                    grad=rng.choice(("f32", dtype, "bf16")), bits=rng.choice((8, 32)))
    if kind == "logprobs":
        vocab = _log(rng, 2, 131_072)
        return dict(kind=kind, rows=_log(rng, 1, min(307_200, 268_435_456 // vocab)), vocab=vocab,
                    top=_log(rng, 1, min(vocab, 64)), dtype=dtype, temperature=rng.choice((0.5, 1.0, 2.0)),
                    mode=rng.choice(("score", "step", "apart")), masked=rng.choice((0.0, 0.1)),
                    blocked=rng.choice((0.0, 0.01)))
    if kind == "quantize4":
        cols = _log(rng, 1, 16384)
        return dict(kind=kind, rows=_log(rng, 1, min(131_072, 67_108_864 // cols)), cols=cols, dtype=dtype)
    # rows, columns and depth of layers from a few labels to a wide one, at most the largest listed product's work
    m, n, k = _log(rng, 1, 307_200), _log(rng, 1, 32768), _log(rng, 16, 8192)
    n = max(1, min(n, 67_108_864 // m, 67_108_864 // k))
    k = max(1, min(k, 67_108_864 // m, 8192**3 // (m * n)))
    c = dict(kind=kind, m=m, n=n, k=k)
    return dict(c, dtype=dtype) if kind == "matmul4" else dict(c, dtype=dtype, out=rng.choice(("f32", "bf16", "f16")))


def _sizes(c):
    """Sizes of the tensors of a step: from the largest down to single values, in no order."""
    n = c["tensors"]
    return [max(1, int(c["largest"] * ((7 * i + n - 1) % n + 1) ** 3 / n**3)) for i in range(n)]


def _held(size):
    return -(-size // HELD) * HELD


RATES = dict(learning_rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.01)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype="f32"):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(DTYPES[dtype])

    s = dict(case=dict(c))
    if c["kind"] == "adamw":
        # the tensors of one buffer, each at a multiple of 128 values; zeros between them
        sizes = _sizes(c)
        spans = [_held(size) for size in sizes]
        starts = [sum(spans[:i]) for i in range(len(spans))]
        at, span = sum(spans), torch.tensor(spans, device="cuda")
        place = torch.arange(at, device="cuda") - torch.repeat_interleave(torch.tensor(starts, device="cuda"), span)
        used = place < torch.repeat_interleave(torch.tensor(sizes, device="cuda"), span)
        # gradients and moments whose sizes differ from tensor to tensor and from value to value, in the midst of a training
        size = torch.exp(normal(at) + torch.repeat_interleave(2 * normal(len(spans)), span) - 7)
        param, grad = normal(at, scale=0.02), normal(at) * size
        first = (0.3 * normal(at) + 0.1 * grad / size) * size
        second = size * size * (0.5 + torch.rand(at, generator=g, device="cuda"))
        param, grad, first, second = (torch.where(used, t, 0.0) for t in (param, grad, first, second))
        param, grad = param.to(DTYPES[c["param"]]), grad.to(DTYPES[c["grad"]])
        s.update(param=param, grad=grad, first=first, second=second, step=100)
        if own:  # the optimizer that a program keeps
            from gsx_amd.backend import AdamW

            s["optimizer"] = AdamW([dict(parameters=[param[a: a + n] for a, n in zip(starts, sizes)],
                                         gradients=[grad[a: a + n] for a, n in zip(starts, sizes)], **RATES)], bits=c["bits"])
            s["optimizer"].load(first, second, steps=100)
        if c["bits"] == 8:
            s["first"], s["second"] = _held_first(first), _held_second(second)
        return s
    if c["kind"] == "logprobs":
        rows, vocab = c["rows"], c["vocab"]
        z = normal(rows, vocab, scale=1.5)
        ids = torch.randint(vocab, (rows,), generator=g, device="cuda")
        if c["blocked"]:  # closed by a mask; the given labels stay open
            z[torch.rand(rows, vocab, generator=g, device="cuda") < c["blocked"]] = -math.inf
        z.scatter_(1, ids[:, None], 3 + 2 * normal(rows, 1))  # a field on its way
        ids = ids.int()
        if c["masked"]:  # rows without a label
            ids[torch.rand(rows, generator=g, device="cuda") < c["masked"]] = -1
        s.update(z=z.to(DTYPES[c["dtype"]]), ids=ids, row_grad=(torch.rand(rows, generator=g, device="cuda") - 1.2) / rows,
                 entropy_grad=torch.rand(rows, generator=g, device="cuda") * 0.01 / rows)
        return s
    if c["kind"] == "quantize4":
        s.update(x=normal(c["rows"], c["cols"], scale=c["cols"] ** -0.5, dtype=c["dtype"]))
        return s
    # features whose channels differ in size, as they do behind a trained layer
    x = normal(c["m"], c["k"]) * torch.exp(normal(c["k"]))
    values, exponents = _quantize4(normal(c["n"], c["k"], scale=c["k"] ** -0.5))
    if c["kind"] == "matmul4":
        s.update(zip(("a_values", "a_exponents"), _quantize4(x.to(DTYPES[c["dtype"]]))))
    else:
        s.update(x=x.to(DTYPES[c["dtype"]]))
    s.update(values=values, exponents=exponents)
    return s


def work(case):
    c = case
    if c["kind"] == "adamw":
        n, blocks = sum(_sizes(c)), sum(_held(size) // HELD for size in _sizes(c))
        step = 2 * BYTES[c["param"]] + BYTES[c["grad"]]
        # 8 bits: codes in, codes out, and the values that they stand for
        states = 16 * n if c["bits"] == 32 else (4 + 8) * n + 16 * blocks
        return dict(bytes=step * n + states, flops=16 * n)
    if c["kind"] == "logprobs":
        b, n = BYTES[c["dtype"]], c["rows"]
        return dict(bytes=n * c["vocab"] * b * (1 if c["mode"] == "score" else 2) + n * c["top"] * 8 + 12 * n,
                    flops=(6 if c["mode"] == "score" else 9) * n * c["vocab"])
    if c["kind"] == "quantize4":
        n = c["rows"] * c["cols"]
        return dict(bytes=n * BYTES[c["dtype"]] + n // 2 + n // BLOCK + 4 * n, flops=2 * n)
    m, n, k = c["m"], c["n"], c["k"]
    x = m * k * BYTES[c["dtype"]] if c["kind"] == "linear4" else m * k // 2 + m * k // BLOCK
    out = BYTES[c["out"]] if c["kind"] == "linear4" else 4
    return dict(bytes=x + n * k // 2 + n * k // BLOCK + m * n * out, flops=2 * m * n * k)


# ---- the plain forms: elementary operations in float32 -----------------------------------------------------------------


def _held_first(m):
    """Blocks of 128 first moments: E4M3 values (kept in their type) and a scale each, float32 numbers all of them."""
    m = m.view(-1, HELD)
    scale = (m.abs().amax(1) * (1 / 448)).clamp(min=2.0**-126)
    return (m * (1 / scale)[:, None]).to(torch.float8_e4m3fn), scale


def _held_second(v):
    """Blocks of 128 second moments: the largest of each and the others' ratio to it, rounded to three bits behind the first
    (ties to even); the least ratio is 2^-32 with the bits 011 behind it. Codes count the ratios upwards, 0 stands for 0."""
    v = v.view(-1, HELD)
    scale = v.amax(1).clamp(min=2.0**-126)
    bits = (v * (1 / scale)[:, None]).view(torch.int32)
    code = ((bits + 0x7FFFF + ((bits >> 20) & 1)) >> 20) - 762
    return torch.where(v > 0, code.clamp(1, 254), 0).to(torch.uint8), scale


def _first_values(held):
    codes, scale = held
    return (codes.float() * scale[:, None]).view(-1)


def _second_values(held):
    codes, scale = held
    ratio = torch.where(codes > 0, (codes.int() + 762) << 20, 0).view(torch.float32)
    return (ratio * scale[:, None]).view(-1)


def _plain_adamw(s):
    c, r = s["case"], RATES
    s["step"] += 1
    b1, b2, lr = r["beta1"], r["beta2"], r["learning_rate"]
    held = c["bits"] == 8
    g = s["grad"].float()
    m = _first_values(s["first"]) if held else s["first"]
    v = _second_values(s["second"]) if held else s["second"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    p = s["param"].float()
    change = m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** s["step"])) + r["epsilon"])
    p = p - lr * r["weight_decay"] * p - lr / (1 - b1 ** s["step"]) * change
    s["param"].copy_(p)
    s["first"], s["second"] = (_held_first(m), _held_second(v)) if held else (m, v)
    if held:
        return dict(param=s["param"], first=_first_values(s["first"]), second=_second_values(s["second"]))
    return dict(param=s["param"], first=m, second=v)


def _ordered(z):
    """Whole numbers that order logits as the top entries are: the larger logit first, of equal ones the lowest index."""
    bits = (z + 0.0).view(torch.int32)
    ordered = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    return (ordered << 32) | (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))


def _plain_logprobs(s):
    c = s["case"]
    z, ids, t = s["z"].float(), s["ids"].long(), c["temperature"]
    known = ids >= 0
    y = z / t
    y = y - y.amax(1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    log_q = y - torch.log(total)
    q = e / total
    open_ = z > -math.inf
    entropy = -torch.where(open_, q * log_q, 0.0).sum(1)
    chosen = torch.where(known, log_q.gather(1, torch.where(known, ids, 0)[:, None])[:, 0], 0.0)
    top = 0xFFFFFFFF - (_ordered(z).topk(c["top"], dim=1).values & 0xFFFFFFFF)
    top_log = log_q.gather(1, top)
    top = torch.where(top_log > -math.inf, top, -1).int()
    out = dict(chosen=chosen, entropy=entropy, top=top, top_log=top_log)
    if c["mode"] == "score":
        return out
    gl = torch.where(known, s["row_grad"], 0.0)[:, None]
    grad = -gl * q
    if c["mode"] == "apart":
        grad = grad - s["entropy_grad"][:, None] * torch.where(open_, q * (log_q + entropy[:, None]), 0.0)
    grad.scatter_add_(1, torch.where(known, ids, 0)[:, None], gl)
    return dict(out, grad=(grad / t).to(s["z"].dtype))


def _power(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _quantize4(x):
    """Rows of x in blocks of 32: two values a byte, the first one low (E2M1: a sign and the place in VALUES4; rows of whole
    blocks), and exponents (e + 127; blocks rounded up to 4)."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    top = x.abs().amax(2)
    half, e = torch.frexp(top)  # top = half * 2^e, half in [0.5, 1); 6 = 0.75 * 2^3
    e = torch.where(top > 0, (e - 3 + (half > 0.75).int()).clamp(min=-100), 0).int()
    y = x * _power(-e)[..., None]
    size = y.abs()
    # halves up to 2, whole numbers up to 4, even ones up to 6, ties to the even place
    wide = torch.where(size < 4, torch.round(size) + 2, torch.round(size / 2) + 4)
    place = torch.where(size < 2, torch.round(2 * size), wide)
    place = (place.int() + 8 * torch.signbit(y).int()).view(rows, blocks * BLOCK // 2, 2)
    exponents = torch.zeros(rows, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    exponents[:, :blocks] = (e + 127).to(torch.uint8)
    return (place[..., 0] + 16 * place[..., 1]).to(torch.uint8), exponents


def _values4(values, exponents, cols):
    """What 4-bit blocks stand for, in float32."""
    sizes = torch.tensor(VALUES4, device=values.device)
    table = torch.cat([sizes, -sizes])
    v = torch.stack([table[(values & 15).long()], table[(values >> 4).long()]], -1).view(values.shape[0], -1, BLOCK)
    return (v * _power(exponents[:, : v.shape[1]].int() - 127)[..., None]).view(values.shape[0], -1)[:, :cols]


def _plain_quantize4(s):
    return _values4(*_quantize4(s["x"]), s["case"]["cols"])


def _plain_matmul4(s):
    k = s["case"]["k"]
    return _values4(s["a_values"], s["a_exponents"], k) @ _values4(s["values"], s["exponents"], k).T


def _plain_linear4(s):
    c = s["case"]
    x = _values4(*_quantize4(s["x"]), c["k"])
    return (x @ _values4(s["values"], s["exponents"], c["k"]).T).to(DTYPES[c["out"]])


# ---- the framework's calls -----------------------------------------------------------------------------------------------


def _own(s):
    from gsx_amd import fields

    c = s["case"]
    if c["kind"] == "adamw":
        s["optimizer"].step()
        first, second = s["optimizer"].moments()
        return dict(param=s["param"], first=first, second=second)
    if c["kind"] == "logprobs":
        how = dict(temperature=c["temperature"])
        if c["mode"] == "step":
            r = fields.log_probs(s["z"], s["ids"], c["top"], grad_scale=1.0, row_grad=s["row_grad"], **how)
            return dict(chosen=r.chosen, entropy=r.entropy, top=r.top_ids, top_log=r.top_log_probs, grad=r.grad)
        r = fields.log_probs(s["z"], s["ids"], c["top"], **how)
        out = dict(chosen=r.chosen, entropy=r.entropy, top=r.top_ids, top_log=r.top_log_probs)
        if c["mode"] == "score":
            return out
        return dict(out, grad=fields.log_probs_backward(s["z"], r.row_stats, s["ids"], s["row_grad"], s["entropy_grad"], **how))
    if c["kind"] == "quantize4":
        return fields.quantize4(s["x"]).float()
    weight = fields.Blocks4(s["values"], s["exponents"], c["k"])
    if c["kind"] == "matmul4":
        return fields.matmul(fields.Blocks4(s["a_values"], s["a_exponents"], c["k"]), weight)
    return fields.linear(s["x"], weight, out_dtype=DTYPES[c["out"]])


def run(state):
    if own:
        return _own(state)
    plain = dict(adamw=_plain_adamw, logprobs=_plain_logprobs, quantize4=_plain_quantize4, matmul4=_plain_matmul4,
                 linear4=_plain_linear4)
    return plain[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def _exact_ratio(code):
    """A second moment's ratio, field by field: code 254 is 1, eight steps a power of two below it."""
    at = (code.long() + 2).double()  # 254 + 2 = 32 * 8
    octave = torch.floor(at / 8)
    return torch.where(code > 0, torch.exp2(octave - 32) * (1 + (at - 8 * octave) / 8), 0.0)


def _exact_step_of(size, bits, least):
    """Distance of the numbers with `bits` behind the first one at `size`."""
    e = torch.floor(torch.log2(torch.where(size > 0, size, 1.0)))
    e = torch.where(torch.exp2(e) > size, e - 1, e)  # whatever the logarithm was rounded to
    e = torch.where(torch.exp2(e + 1) <= size, e + 1, e)
    return torch.exp2(e.clamp(min=least) - bits)


def _single(x):
    """x rounded to 32 bits."""
    return x.float().double()


def _exact_held(m, v, g):
    """Moments after a step, held in 8 bits. What is held are float32 numbers: each product and sum that leads to one is
    rounded, and so are a block's scale, its inverse and the ratios to it, whose codes are then the nearest ones."""
    r = RATES
    kept, new = (_single(torch.tensor([b, 1 - b], dtype=torch.float64, device="cuda")) for b in (r["beta1"], r["beta2"]))
    m = _single(_single(kept[0] * m) + _single(kept[1] * g)).view(-1, HELD)
    v = _single(_single(new[0] * v) + _single(new[1] * _single(g * g))).view(-1, HELD)
    scale = _single(m.abs().amax(1, keepdim=True) * _single(torch.tensor(1 / 448, dtype=torch.float64, device="cuda")))
    scale = scale.clamp(min=2.0**-126)
    m = _single(m * _single(1 / scale))
    step = _exact_step_of(m.abs(), 3, -6)
    m = (torch.round(m / step) * step).clamp(-448, 448) * scale
    scale = v.amax(1, keepdim=True).clamp(min=2.0**-126)
    ratio = _single(v * _single(1 / scale))
    step = _exact_step_of(ratio, 3, -40)
    ratio = (torch.round(ratio / step) * step).clamp(min=2.0**-32 * 1.375)
    return m.view(-1), (torch.where(v > 0, ratio, 0.0) * scale).view(-1)


def _exact_adamw(s):
    c, r = s["case"], RATES
    g = s["grad"].double()
    if c["bits"] == 8:
        m = _single((s["first"][0].double() * s["first"][1].double()[:, None]).view(-1))
        v = _single((_exact_ratio(s["second"][0]) * s["second"][1].double()[:, None]).view(-1))
        held = _exact_held(m, v, g)
    else:
        m, v = s["first"].double(), s["second"].double()
        held = None
    m = torch.lerp(g, m, r["beta1"])
    v = torch.lerp(g.square(), v, r["beta2"])
    t = s["step"] + 1
    p = s["param"].double()
    new = p * (1 - r["learning_rate"] * r["weight_decay"])
    new -= r["learning_rate"] * (m / (1 - r["beta1"] ** t)) / ((v / (1 - r["beta2"] ** t)).sqrt() + r["epsilon"])
    return dict(param=new, first=m if held is None else held[0], second=v if held is None else held[1])


def _exact_logprobs(s):
    c = s["case"]
    rows, vocab, t = c["rows"], c["vocab"], c["temperature"]
    chosen, entropy = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    top = torch.zeros(rows, c["top"], dtype=torch.int32, device="cuda")
    top_log = torch.zeros(rows, c["top"], dtype=torch.float64, device="cuda")
    grad = None if c["mode"] == "score" else torch.zeros(rows, vocab, dtype=torch.float64, device="cuda")
    part = max(1, 33_554_432 // vocab)
    for at in range(0, rows, part):
        r = slice(at, at + part)
        z, ids = s["z"][r].double(), s["ids"][r].long()
        log_q = torch.log_softmax(z / t, 1)
        q = log_q.exp()
        entropy[r] = torch.special.entr(q).sum(1)
        known = ids >= 0
        at_id = ids.clamp(min=0)[:, None]
        chosen[r] = torch.where(known, log_q.gather(1, at_id)[:, 0], 0.0)
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : c["top"]]
        top_log[r] = log_q.gather(1, order)
        top[r] = torch.where(top_log[r] > -math.inf, order, -1).int()
        if grad is None:
            continue
        gl = torch.where(known, s["row_grad"][r].double(), 0.0)[:, None]
        row = -gl * q
        row.scatter_add_(1, at_id, gl)
        if c["mode"] == "apart":
            row += s["entropy_grad"][r].double()[:, None] * (torch.special.entr(q) - q * entropy[r][:, None])
        grad[r] = row / t
    out = dict(chosen=chosen, entropy=entropy, top=top, top_log=top_log)
    return out if grad is None else dict(out, grad=grad)


def _exact_rounded4(x):
    """x as blocks of 32 along its rows stand for it: the nearest of the 15 values times a power of two that brings the block's
    largest to 6 or less."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], BLOCK * 64):
        v = x[:, at: at + BLOCK * 64].double()
        cols = v.shape[1]
        v = torch.nn.functional.pad(v, (0, -cols % BLOCK)).view(v.shape[0], -1, BLOCK)
        top = v.abs().amax(2, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 6.0) / 6)).clamp(min=-100))
        scale = torch.where(top > 6 * scale, 2 * scale, scale)  # whatever the logarithm was rounded to
        scale = torch.where((top > 0) & (top <= 3 * scale) & (scale > 2.0**-100), scale / 2, scale)
        v = v / scale
        step = _exact_step_of(v.abs(), 1, 0)
        out[:, at: at + cols] = (torch.round(v / step) * step * scale).view(v.shape[0], -1)[:, :cols]
    return out


def _exact_values4(values, exponents, cols):
    """4-bit values and exponents, read field by field."""
    b = torch.stack([values & 15, values >> 4], -1).view(values.shape[0], -1).long()
    field, low = (b >> 1) & 3, (b & 1).double()
    v = torch.where(field == 0, low / 2, (1 + low / 2) * torch.exp2(field.double() - 1))
    v = torch.where(b > 7, -v, v)
    return (v * torch.exp2(exponents.double() - 127).repeat_interleave(BLOCK, 1)[:, : v.shape[1]])[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["case"]["kind"]
    if kind == "adamw":
        return _exact_adamw(s)
    if kind == "logprobs":
        return _exact_logprobs(s)
    if kind == "quantize4":
        return _exact_rounded4(s["x"])
    k = s["case"]["k"]
    a = _exact_rounded4(s["x"]) if kind == "linear4" else _exact_values4(s["a_values"], s["a_exponents"], k)
    return a @ _exact_values4(s["values"], s["exponents"], k).T
