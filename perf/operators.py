"""Performance cases of the label-field operators: rows looked up by code, a head in 8-bit blocks, and a loss against a
teacher's top logits.

A label field attaches a code (a token id) to each Gaussian or pixel. A training step looks the codes' rows up, multiplies
them with a head whose weights are held as 8-bit blocks, compares the logits with the top logits of a large teacher, and
carries the gradient back through head and lookup; a query of a trained field is the same path for one row. A case is one
pass through one operator:

  lookup       rows of a table by id, scaled
  lookup_grad  the table's gradient: the rows' gradients summed by id
  linear       rows quantised to 8-bit blocks of 128 and multiplied with a weight held so
  linear_grad  both gradients of that product, their operands quantised the same way
  distill      the loss against a teacher's top logits: with its gradient in one pass ("step"), alone ("loss"), or with the
               gradient in a later call, from upstream gradients ("apart")

`run` computes them in elementary float32 torch operations, or with gsx_amd.fields where `own` is true.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128


def listed():
    return [
        # one token's row for a single query: what a call costs
        dict(name="lookup_token", kind="lookup", count=1, table_rows=65536, width=4096, dtype="bf16", skew=1, masked=0.0),
        # the codes of the 1M Gaussians of the benchmark scene in a codebook of 8192 rows; a tenth have none
        dict(name="lookup_codebook", kind="lookup", count=1_000_000, table_rows=8192, width=64, dtype="f32", skew=4,
             masked=0.1),
        # a short training text against a small table, odd sizes
        dict(name="lookup_grad_small", kind="lookup_grad", count=77, table_rows=1001, width=385, dtype="f32", skew=2,
             masked=0.0),
        # the codebook's gradient: 1M rows on 8192, the most frequent code drawn by a tenth of them
        dict(name="lookup_grad_codebook", kind="lookup_grad", count=1_000_000, table_rows=8192, width=64, dtype="f32",
             skew=4, masked=0.1),
        # a batch of 16384 tokens on a whole vocabulary: most rows of the gradient are zeros to be written
        dict(name="lookup_grad_vocab", kind="lookup_grad", count=16384, table_rows=65536, width=2048, dtype="bf16", skew=2,
             masked=0.0),
        # the logits of one query: a weight of 128 MB read for a single row
        dict(name="linear_token", kind="linear", m=1, n=32768, k=4096, dtype="bf16", out="f32"),
        # a head of 150 labels on the pixels of a 640x480 frame of 128 features
        dict(name="linear_pixels", kind="linear", m=307_200, n=150, k=128, dtype="bf16", out="bf16"),
        # a batch of 8192 rows through a wide square layer
        dict(name="linear_large", kind="linear", m=8192, n=8192, k=8192, dtype="bf16", out="bf16"),
        # the label head's gradients: one of them sums over all 307200 pixels
        dict(name="linear_grad_pixels", kind="linear_grad", m=307_200, n=150, k=128, dtype="bf16"),
        # gradients of a layer on a batch with odd sizes
        dict(name="linear_grad_odd", kind="linear_grad", m=4001, n=4100, k=2050, dtype="f32"),
        # a teacher's 64 top logits against one row of a large vocabulary
        dict(name="distill_token", kind="distill", rows=1, vocab=131072, top=64, dtype="f32", temperature=2.0, mode="step",
             masked=0.0, blocked=0.0),
        # a batch against an odd vocabulary; a part of the rows is padding, some logits are closed by a mask
        dict(name="distill_vocab", kind="distill", rows=4096, vocab=65537, top=64, dtype="bf16", temperature=2.0,
             mode="step", masked=0.1, blocked=0.01),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("lookup", "lookup_grad", "linear", "linear_grad", "distill"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if kind in ("lookup", "lookup_grad"):
        width = _log(rng, 1, 4096)
        return dict(kind=kind, count=_log(rng, 1, min(1_000_000, 64_000_000 // width)),
                    table_rows=_log(rng, 1, min(131_072, 134_217_728 // width)), width=width, dtype=dtype,
                    skew=rng.choice((1, 2, 4)), masked=rng.choice((0.0, 0.1)))
    if kind in ("linear", "linear_grad"):
        # rows, columns and depth of layers from a few labels to a wide one, at most the largest listed product's work
        most = 8192**3 if kind == "linear" else 8192**3 // 4
        m, n, k = _log(rng, 1, 307_200), _log(rng, 1, 32768), _log(rng, 16, 8192)
        n = max(1, min(n, 67_108_864 // m, 67_108_864 // k))
        k = max(1, min(k, 67_108_864 // m, most // (m * n)))
        c = dict(kind=kind, m=m, n=n, k=k, dtype=dtype)
        return dict(c, out=rng.choice(("f32", "bf16", "f16"))) if kind == "linear" else c
    vocab = _log(rng, 2, 131_072)
    return dict(kind=kind, rows=_log(rng, 1, min(307_200, 268_435_456 // vocab)), vocab=vocab,
                top=_log(rng, 1, min(vocab, 256)), dtype=dtype, temperature=rng.choice((0.5, 1.0, 2.0)),
                mode=rng.choice(("step", "loss", "apart")), masked=rng.choice((0.0, 0.1)), blocked=rng.choice((0.0, 0.01)))


def _ids(g, c):
    """Ids with the given skew (the most frequent one has a share of table_rows^(-1/skew)); -1 for rows without a code."""
    u = torch.rand(c["count"], generator=g, device="cuda", dtype=torch.float64)
    ids = (u ** c["skew"] * c["table_rows"]).long().clamp_(max=c["table_rows"] - 1).int()
    if c["masked"]:
        ids[torch.rand(c["count"], generator=g, device="cuda") < c["masked"]] = -1
    return ids


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype="f32"):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(DTYPES[dtype])

    s = dict(case=dict(c))
    if c["kind"] == "lookup":
        s.update(table=normal(c["table_rows"], c["width"], dtype=c["dtype"]), ids=_ids(g, c), scale=math.sqrt(c["width"]))
    elif c["kind"] == "lookup_grad":
        s.update(grad=normal(c["count"], c["width"], scale=1e-3, dtype=c["dtype"]), ids=_ids(g, c),
                 scale=math.sqrt(c["width"]))
    elif c["kind"] == "linear":
        # features whose channels differ in size, as they do behind a trained layer
        x = normal(c["m"], c["k"]) * torch.exp(normal(c["k"]))
        values, exponents = _quantize(normal(c["n"], c["k"], scale=c["k"] ** -0.5))
        s.update(x=x.to(DTYPES[c["dtype"]]), values=values, exponents=exponents)
    elif c["kind"] == "linear_grad":
        x = normal(c["m"], c["k"]) * torch.exp(normal(c["k"]))
        values, exponents = _quantize(normal(c["k"], c["n"], scale=c["k"] ** -0.5))  # the transposed weight
        s.update(x=x.to(DTYPES[c["dtype"]]), grad=normal(c["m"], c["n"], scale=1e-4, dtype=c["dtype"]), values=values,
                 exponents=exponents)
    else:
        rows, vocab, top = c["rows"], c["vocab"], c["top"]
        # the teacher's top entries: one of each of `top` equal parts of the vocabulary, the largest logits first
        part = vocab // top
        ids = torch.randint(part, (rows, top), generator=g, device="cuda") + part * torch.arange(top, device="cuda")
        teacher = (normal(rows, top, scale=1.5) + 4).sort(dim=1, descending=True).values
        z = normal(rows, vocab, scale=1.5)
        if c["blocked"]:  # closed by a mask; the teacher's entries stay open
            z[torch.rand(rows, vocab, generator=g, device="cuda") < c["blocked"]] = -math.inf
        z.scatter_(1, ids, 0.7 * teacher + normal(rows, top))  # a student on its way
        weight = torch.rand(rows, generator=g, device="cuda") + 0.5
        ids = ids.int()
        if c["masked"]:  # padding rows, and rows whose teacher names fewer entries
            weight[torch.rand(rows, generator=g, device="cuda") < c["masked"]] = 0
            ids[torch.rand(rows, top, generator=g, device="cuda") < c["masked"]] = -1
        upstream = torch.rand(rows, generator=g, device="cuda") / rows
        s.update(z=z.to(DTYPES[c["dtype"]]), ids=ids, teacher=teacher, weight=weight, upstream=upstream)
    return s


def work(case):
    c = case
    if c["kind"] in ("lookup", "lookup_grad"):
        b, n, w = BYTES[c["dtype"]], c["count"], c["width"]
        if c["kind"] == "lookup":
            return dict(bytes=4 * n + min(n, c["table_rows"]) * w * b + n * w * b, flops=n * w)
        return dict(bytes=4 * n + n * w * b + 4 * c["table_rows"] * w, flops=2 * n * w)
    if c["kind"] in ("linear", "linear_grad"):
        b, m, n, k = BYTES[c["dtype"]], c["m"], c["n"], c["k"]
        weight = n * k + n * k // BLOCK
        if c["kind"] == "linear":
            return dict(bytes=m * k * b + weight + m * n * BYTES[c["out"]], flops=2 * m * n * k)
        return dict(bytes=2 * m * k * b + m * n * b + weight + 4 * n * k, flops=4 * m * n * k)
    b, n = BYTES[c["dtype"]], c["rows"]
    return dict(bytes=n * c["vocab"] * b * (1 if c["mode"] == "loss" else 2) + n * c["top"] * 8 + 8 * n,
                flops=(4 if c["mode"] == "loss" else 6) * n * c["vocab"])


# ---- the plain forms: elementary operations in float32 -----------------------------------------------------------------


def _power(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _quantize(x):
    """Rows of x in blocks of 128: values (E4M3 bytes, [rows, columns rounded up to 128]) and exponents (e + 127, [rows, blocks
    rounded up to 4])."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    top = x.abs().amax(2)
    half, e = torch.frexp(top)  # top = half * 2^e, half in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, (e - 9 + (half > 0.875).int()).clamp(min=-100), 0).int()
    values = (x * _power(-e)[..., None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK).view(torch.uint8)
    exponents = torch.zeros(rows, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    exponents[:, :blocks] = (e + 127).to(torch.uint8)
    return values, exponents


def _values(values, exponents, cols):
    """What blocks stand for, in float32."""
    blocks = values.shape[1] // BLOCK
    x = values.view(torch.float8_e4m3fn).float().view(-1, blocks, BLOCK)
    return (x * _power(exponents[:, :blocks].int() - 127)[..., None]).view(-1, blocks * BLOCK)[:, :cols]


def _rounded(x):
    return _values(*_quantize(x), x.shape[1])


def _plain_lookup(s):
    table, ids = s["table"], s["ids"].long()
    fits = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(fits, ids, 0)].float() * s["scale"]
    return torch.where(fits[:, None], rows, 0.0).to(table.dtype)


def _plain_lookup_grad(s):
    ids, rows = s["ids"].long(), s["case"]["table_rows"]
    fits = (ids >= 0) & (ids < rows)
    grad = torch.where(fits[:, None], s["grad"].float(), 0.0) * s["scale"]
    return torch.zeros(rows, grad.shape[1], device="cuda").index_add_(0, torch.where(fits, ids, 0), grad)


def _plain_linear(s):
    c = s["case"]
    return (_rounded(s["x"]) @ _values(s["values"], s["exponents"], c["k"]).T).to(DTYPES[c["out"]])


def _plain_linear_grad(s):
    c = s["case"]
    grad_x = _rounded(s["grad"]) @ _values(s["values"], s["exponents"], c["n"]).T
    grad_w = _rounded(s["grad"].T) @ _rounded(s["x"].T).T
    return dict(x=grad_x.to(DTYPES[c["dtype"]]), weight=grad_w)


def _plain_distill(s):
    c = s["case"]
    t, vocab = c["temperature"], c["vocab"]
    ids = s["ids"].long()
    fits = (ids >= 0) & (ids < vocab) & (s["teacher"] > -math.inf)
    ids = torch.where(fits, ids, 0)
    teacher = torch.where(fits, s["teacher"] / t, -math.inf)
    some = fits.any(1) & (s["weight"] != 0)
    teacher = teacher - torch.where(some, teacher.amax(1), 0.0)[:, None]
    p = torch.where(fits, torch.exp(teacher), 0.0)
    total = p.sum(1, keepdim=True)
    log_p = teacher - torch.log(total)
    p = p / torch.where(total > 0, total, 1.0)
    z = s["z"].float() / t
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    log_q = z.gather(1, ids) - lse
    loss = torch.where(some, s["weight"] * t * t * torch.where(fits, p * (log_p - log_q), 0.0).sum(1), 0.0)
    if c["mode"] == "loss":
        return dict(loss=loss)
    grad = (e / total).scatter_add_(1, ids, -p)
    scale = s["upstream"] if c["mode"] == "apart" else 1.0 / c["rows"]
    grad = torch.where(some[:, None], grad * (s["weight"] * scale * t)[:, None], 0.0)
    return dict(loss=loss, grad=grad.to(s["z"].dtype))


# ---- the framework's calls -----------------------------------------------------------------------------------------------


def _own(s):
    from gsx_amd import fields

    c = s["case"]
    if c["kind"] == "lookup":
        return fields.lookup(s["table"], s["ids"], scale=s["scale"])
    if c["kind"] == "lookup_grad":
        return fields.lookup_backward(s["grad"], s["ids"], c["table_rows"], scale=s["scale"])
    if c["kind"] == "linear":
        weight = fields.Blocks(s["values"], s["exponents"], c["k"])
        return fields.linear(s["x"], weight, out_dtype=DTYPES[c["out"]])
    if c["kind"] == "linear_grad":
        weight = fields.Blocks(s["values"], s["exponents"], c["n"])
        grad_x, grad_w = fields.linear_backward(s["x"], s["grad"], weight)
        return dict(x=grad_x, weight=grad_w)
    how = dict(temperature=c["temperature"], row_weight=s["weight"])
    if c["mode"] == "step":
        loss, _, grad = fields.distill(s["z"], s["ids"], s["teacher"], grad_scale=1.0 / c["rows"], **how)
        return dict(loss=loss, grad=grad)
    loss, lse, _ = fields.distill(s["z"], s["ids"], s["teacher"], **how)
    if c["mode"] == "loss":
        return dict(loss=loss)
    return dict(loss=loss, grad=fields.distill_backward(s["z"], lse, s["ids"], s["teacher"], s["upstream"], **how))


def run(state):
    if own:
        return _own(state)
    plain = dict(lookup=_plain_lookup, lookup_grad=_plain_lookup_grad, linear=_plain_linear,
                 linear_grad=_plain_linear_grad, distill=_plain_distill)
    return plain[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def _exact_rounded(x):
    """x as blocks of 128 along its rows stand for it: E4M3 steps of a power of two that brings the block's largest value to
    448 or less."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], BLOCK):
        v = x[:, at: at + BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448)).clamp(min=-100))
        scale = torch.where(top > 448 * scale, 2 * scale, scale)  # whatever the logarithm was rounded to
        scale = torch.where((top > 0) & (top <= 224 * scale) & (scale > 2.0**-100), scale / 2, scale)
        v = v / scale
        size = torch.where(v == 0, 1.0, v.abs())
        step = torch.exp2(torch.floor(torch.log2(size)).clamp(min=-6) - 3)
        # just below a power of two the logarithm may round up to it; the finer step is the right one there
        step = torch.where((size < 8 * step) & (step > 2.0**-9), step / 2, step)
        out[:, at: at + BLOCK] = torch.round(v / step) * step * scale
    return out


def _exact_values(s, cols):
    """E4M3 bytes and exponents, read field by field."""
    b = s["values"].long()
    field, low = (b >> 3) & 15, (b & 7).double()
    v = torch.where(field == 0, low * 2.0**-9, (1 + low / 8) * torch.exp2(field.double() - 7))
    v = torch.where(b > 127, -v, v)
    e = torch.exp2(s["exponents"].double() - 127).repeat_interleave(BLOCK, 1)[:, : v.shape[1]]
    return (v * e)[:, :cols]


def _exact_linear(s):
    return _exact_rounded(s["x"]) @ _exact_values(s, s["case"]["k"]).T


def _exact_linear_grad(s):
    return dict(x=_exact_rounded(s["grad"]) @ _exact_values(s, s["case"]["n"]).T,
                weight=_exact_rounded(s["grad"].T.contiguous()) @ _exact_rounded(s["x"].T.contiguous()).T)


def _exact_lookup(s):
    table = torch.cat([s["table"].double() * s["scale"], torch.zeros(1, s["table"].shape[1], device="cuda")])
    return table[s["ids"].long()]  # -1, no code, is the row of zeros at the end


def _exact_lookup_grad(s):
    out = torch.zeros(s["case"]["table_rows"] + 1, s["case"]["width"], dtype=torch.float64, device="cuda")
    out.index_add_(0, torch.where(s["ids"] < 0, out.shape[0] - 1, s["ids"].long()), s["grad"].double())
    return out[:-1] * s["scale"]


def _exact_distill(s):
    c = s["case"]
    t, upstream = c["temperature"], s["upstream"] if c["mode"] == "apart" else torch.full_like(s["upstream"], 1.0 / c["rows"])
    loss = torch.zeros(c["rows"], dtype=torch.float64, device="cuda")
    grad = None if c["mode"] == "loss" else torch.zeros(c["rows"], c["vocab"], dtype=torch.float64, device="cuda")
    part = max(1, 33_554_432 // c["vocab"])
    for at in range(0, c["rows"], part):
        r = slice(at, at + part)
        log_q = torch.log_softmax(s["z"][r].double() / t, 1)
        ids = s["ids"][r].long()
        teacher = torch.where(ids < 0, -math.inf, s["teacher"][r].double() / t)
        log_p = torch.log_softmax(teacher, 1).nan_to_num(nan=-math.inf)  # no entry at all: no mass
        p = log_p.exp()
        terms = p * (log_p.clamp(min=-1e300) - log_q.gather(1, ids.clamp(min=0)))
        weight = s["weight"][r].double()
        loss[r] = weight * t * t * torch.where(p > 0, terms, 0.0).sum(1)
        if grad is not None:
            row = log_q.exp() * p.sum(1, keepdim=True)
            row.scatter_add_(1, ids.clamp(min=0), -p)
            grad[r] = row * (weight * upstream[r].double() * t)[:, None]
    return dict(loss=loss) if grad is None else dict(loss=loss, grad=grad)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(lookup=_exact_lookup, lookup_grad=_exact_lookup_grad, linear=_exact_linear,
                linear_grad=_exact_linear_grad, distill=_exact_distill)[case["kind"]](s)
