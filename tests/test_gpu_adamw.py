"""AdamW over many tensors: steps against 64 bits, 8-bit moments bit by bit, counts on the device, streams and graphs."""
import numpy as np
import pytest

import adamw_plain as plain

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
RATES = dict(learning_rate=1e-2, beta1=0.9, beta2=0.999, weight_decay=0.01, epsilon=1e-8)
SIZES = [1, 7, 0, 127, 128, 129, 2047, 2048, 2049, 5000, 3]


def _np(t):
    return t.detach().double().cpu().numpy()


class Case:
    """Tensors of given sizes (lead: elements before each in its memory), moments in the midst of a training."""

    def __init__(self, sizes, param, grad, seed, lead=0):
        rng = np.random.default_rng(seed)
        self.p, self.g, self.m, self.v = [], [], [], []
        for n in sizes:
            def put(x, dtype):
                room = torch.zeros(n + lead, dtype=DTYPES[dtype], device="cuda")
                room[lead:] = torch.from_numpy(x).to("cuda")
                return room[lead:]
            size = np.exp(rng.standard_normal(n) * 2 - 4)
            self.p.append(put(rng.standard_normal(n), param))
            self.g.append(put(rng.standard_normal(n) * size, grad))
            self.m.append((rng.standard_normal(n) * size * 0.3).astype(np.float32))
            self.v.append((size**2 * rng.uniform(0.1, 2, n)).astype(np.float32))

    def optimizer(self, bits, groups=None, steps=0):
        from gsx_amd.backend import AdamW
        opt = AdamW(groups or [dict(parameters=self.p, gradients=self.g, **RATES)], bits=bits)
        m, v = np.zeros(opt.size, np.float32), np.zeros(opt.size, np.float32)
        for at, a, b in zip(opt.offsets, self.m, self.v):
            m[at: at + len(a)], v[at: at + len(b)] = a, b
        opt.load(torch.from_numpy(m).cuda(), torch.from_numpy(v).cuda(), steps)
        return opt


def _rounding(t, size):
    """Half a step of the type of t at values of this size: below the least normal number steps stay what they are there (float16:
    2^-14 has steps of 2^-24, and so have all smaller values)."""
    if t.dtype == torch.float32:
        return 0
    return torch.finfo(t.dtype).eps / 2 * np.maximum(size, torch.finfo(t.dtype).smallest_normal)


def _check(case, opt, before, scale, t, rates=RATES, only=None):
    """Every tensor against the step from `before` (parameters, moments); only: tensors that had one."""
    first, second = (_np(x) for x in opt.moments())
    for i, (p, g) in enumerate(zip(case.p, case.g)):
        p0, m0, v0 = before[i]
        n, at = len(p0), opt.offsets[i]
        if only is not None and i not in only:
            assert np.array_equal(_np(p), p0)
            continue
        want, off = plain.step(p0, _np(g), m0, v0, scale, t, rates)
        got = _np(p)
        assert (np.abs(got - want[0]) <= off[0] + _rounding(p, np.abs(want[0]) + off[0])).all(), i
        if opt.bits == 32:
            assert (np.abs(first[at: at + n] - want[1]) <= off[1]).all(), i
            assert (np.abs(second[at: at + n] - want[2]) <= off[2]).all(), i
        else:
            m1, v1 = plain.moments32(m0.astype(np.float32), v0.astype(np.float32), g.float().cpu().numpy(), scale, rates)
            span = -(-n // 128) * 128
            for hold, new, codes, scales in ((plain.hold_first, m1, opt.first, opt.first_scale),
                                             (plain.hold_second, v1, opt.second, opt.second_scale)):
                q, s = hold(new)
                assert np.array_equal(codes[at: at + span].cpu().numpy(), q), i
                assert np.array_equal(scales[at // 128: (at + span) // 128].cpu().numpy(), s), i
            assert np.array_equal(first[at: at + span], plain.first_values(*plain.hold_first(m1)).astype(np.float64))
            assert np.array_equal(second[at: at + span], plain.second_values(*plain.hold_second(v1)).astype(np.float64))


def _state(case, opt):
    first, second = (_np(x) for x in opt.moments())
    return [(_np(p), first[at: at + p.numel()], second[at: at + p.numel()]) for p, at in zip(case.p, opt.offsets)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", DTYPES)
@pytest.mark.parametrize("param", DTYPES)
def test_steps_against_64_bits(param, grad, bits):
    print(f"[case] adamw {param} {grad} {bits}", flush=True)
    case = Case(SIZES, param, grad, 1)
    opt = case.optimizer(bits, steps=10)
    for t in (11, 12, 13):
        before = _state(case, opt)
        opt.step()
        _check(case, opt, before, 1.0, t)
    assert opt.steps.item() == 13


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32")])
def test_memory_that_is_aligned_to_elements_only(param, grad, bits):
    case = Case(SIZES, param, grad, 2, lead=1)
    opt = case.optimizer(bits)
    before = _state(case, opt)
    opt.step(grad_scale=0.25)
    _check(case, opt, before, 0.25, 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_in_groups_and_a_factor_on_the_device(bits):
    case = Case([(17 * i * i) % 4099 + 1 for i in range(300)], "f32", "f32", 3)
    rates = [dict(RATES, learning_rate=1e-2 / (k + 1), beta1=0.8 + 0.01 * k, beta2=0.99, weight_decay=0.1 * k) for k in range(16)]
    cut = [round(300 * k / 16) for k in range(17)]
    groups = [dict(parameters=case.p[a:b], gradients=case.g[a:b], **r) for a, b, r in zip(cut, cut[1:], rates)]
    opt = case.optimizer(bits, groups)
    before = _state(case, opt)
    factor = torch.tensor([0.5], device="cuda")
    opt.step(grad_scale=0.5, grad_factor=factor)
    for k, r in enumerate(rates):
        part = Case([], "f32", "f32", 0)
        part.p, part.g = case.p[cut[k]: cut[k + 1]], case.g[cut[k]: cut[k + 1]]

        class View:
            pass
        view = View()
        view.__dict__.update(opt.__dict__, offsets=opt.offsets[cut[k]: cut[k + 1]], moments=opt.moments)
        _check(part, view, before[cut[k]: cut[k + 1]], 0.25, 1, r)


def test_a_fresh_optimizer_starts_from_zero_moments():
    for bits in (8, 32):
        case = Case([300], "f32", "f32", 4)
        from gsx_amd.backend import AdamW
        opt = AdamW([dict(parameters=case.p, gradients=case.g, **RATES)], bits=bits)
        before = _state(case, opt)
        assert not before[0][1].any() and not before[0][2].any()
        opt.step()
        _check(case, opt, before, 1.0, 1)


def test_moments_of_special_values_are_held_bit_by_bit():
    from gsx_amd.backend import AdamW
    rng = np.random.default_rng(5)
    n = 128 * 64
    m = (rng.standard_normal(n) * 2.0 ** rng.integers(-20, 20, n)).astype(np.float32)
    v = (rng.random(n) * 2.0 ** rng.integers(-40, 20, n)).astype(np.float32)
    m[::7], v[::7] = 0, 0
    for b, (x, y) in enumerate([(0, 0), (1e-45, 1e-45), (3.4e38, 3.4e38), (1e-38, 1e-38), (-1.0, 1.0)]):
        m[b * 128: b * 128 + 100], v[b * 128: b * 128 + 100] = x, y
    m[1000], m[1001], m[1002], v[1003], v[1004] = np.nan, np.inf, -np.inf, np.inf, np.nan
    m[1280:1408], v[1280:1408] = np.nan, np.inf  # nothing finite in a block
    m[2048:2175], v[2048:2175] = np.arange(127) * 3.5 / 448, np.linspace(0, 1, 127)  # ties, and the largest in the last place
    m[2175], v[2175] = 1.0, 1.0
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt = AdamW([dict(parameters=[p], gradients=[g], **RATES)], bits=8)
    opt.load(torch.from_numpy(m).cuda(), torch.from_numpy(v).cuda(), 5)
    for hold, values, x, codes, scales, back in (
            (plain.hold_first, plain.first_values, m, opt.first, opt.first_scale, opt.moments()[0]),
            (plain.hold_second, plain.second_values, v, opt.second, opt.second_scale, opt.moments()[1])):
        q, s = hold(x)
        assert np.array_equal(scales.cpu().numpy(), s)
        assert np.array_equal(codes.cpu().numpy(), q)
        assert np.array_equal(back.cpu().numpy(), values(q, s), equal_nan=True)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    """NaN and infinite gradients spoil their own elements, not their block's others; one whose square overflows stops its own."""
    case = Case([256], "f32", "f32", 6)
    opt = case.optimizer(bits)
    before = _state(case, opt)
    clean = Case([256], "f32", "f32", 6)
    other = clean.optimizer(bits)
    case.g[0][3], case.g[0][100], case.g[0][200] = float("nan"), float("inf"), 1e30
    clean.g[0][3] = clean.g[0][100] = clean.g[0][200] = 0
    opt.step()
    other.step()
    got, want = _np(case.p[0]), _np(clean.p[0])
    keep = np.ones(256, bool)
    keep[[3, 100, 200]] = False
    assert np.array_equal(got[keep], want[keep])
    assert np.isnan(got[[3, 100]]).all()
    decayed = before[0][0][200] * (1 - RATES["learning_rate"] * RATES["weight_decay"])
    assert abs(got[200] - decayed) <= 3 * 2.0**-24 * abs(decayed)  # m / inf = 0
    opt.step()  # codes of what is not finite lead to the same again
    got = _np(case.p[0])
    assert np.isnan(got[[3, 100]]).all() and np.isfinite(got[200])


def test_a_second_moment_is_never_held_as_zero():
    """A small value beside a large one keeps a denominator: its update stays below the learning rate times m / sqrt(v)'s bound."""
    from gsx_amd.backend import AdamW
    p, g = torch.zeros(128, device="cuda"), torch.full((128,), 1e-7, device="cuda")
    g[0] = 1e3
    opt = AdamW([dict(parameters=[p], gradients=[g], **dict(RATES, weight_decay=0.0))], bits=8)
    for _ in range(20):
        opt.step()
    # sqrt(1 - 0.999) / (1 - 0.9) bounds |m| / sqrt(v) by 3.2, bias corrections by 32 at the first step
    assert p.abs().max().item() <= 20 * RATES["learning_rate"] * 3.2
    assert (opt.second[1:] >= 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_a_captured_step_count_on(bits):
    case, twin = (Case([5000, 33], "bf16", "bf16", 7) for _ in range(2))
    opt, other = case.optimizer(bits), twin.optimizer(bits)
    opt.step()
    other.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grad_scale=0.5)
    for k in range(4):
        for a, b in zip(case.g, twin.g):
            a.mul_(0.9)
            b.mul_(0.9)
        graph.replay()
        other.step(grad_scale=0.5)
        assert opt.steps.item() == other.steps.item() == 2 + k
        for a, b in zip(case.p + [opt.first, opt.second], twin.p + [other.first, other.second]):
            assert torch.equal(a, b)


def test_on_another_stream():
    case, twin = (Case([100_000], "f32", "f32", 8) for _ in range(2))
    opt, other = case.optimizer(8), twin.optimizer(8)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        opt.step(stream=s)
        other.step()
    first, second = opt.moments(stream=s)
    s.synchronize()
    assert torch.equal(case.p[0], twin.p[0])
    want = other.moments()
    assert torch.equal(first, want[0]) and torch.equal(second, want[1])


def test_rates_may_change_between_steps():
    case = Case([1000], "f32", "f32", 9)
    opt = case.optimizer(32)
    for t, lr in ((1, 1e-3), (2, 5e-2)):
        opt.groups[0]["learning_rate"] = lr
        before = _state(case, opt)
        opt.step()
        _check(case, opt, before, 1.0, t, dict(RATES, learning_rate=lr))


def test_a_saved_training_goes_on():
    case, twin = (Case([3000], "f32", "f32", 10) for _ in range(2))
    opt, other = case.optimizer(32), twin.optimizer(32)
    opt.step()
    other.step()
    first, second = (x.clone() for x in opt.moments())
    resumed = case.optimizer(32)
    resumed.load(first, second, int(opt.steps.item()))
    resumed.step()
    other.step()
    assert torch.equal(case.p[0], twin.p[0])


def test_refusals():
    from gsx_amd.backend import AdamW, GsxHipError
    p, g = torch.zeros(10, 4, device="cuda"), torch.zeros(10, 4, device="cuda")
    good = dict(parameters=[p], gradients=[g], learning_rate=1e-3)
    for groups, bits in (([good], 16), ([], 32), ([good] * 17, 32), ([good, good], 32),
                         ([dict(good, gradients=[])], 32), ([dict(good, gradients=[g.cpu()])], 32),
                         ([dict(good, gradients=[g.view(4, 10)])], 32), ([dict(good, gradients=[g.double()])], 32),
                         ([dict(good, parameters=[p.T], gradients=[g.T])], 32), ([dict(good, gradients=[p])], 32)):
        with pytest.raises(GsxHipError):
            AdamW(groups, bits=bits)
    opt = AdamW([good], bits=8)
    for call in (lambda: opt.step(grad_factor=torch.ones(1)), lambda: opt.step(grad_factor=torch.ones(2, device="cuda")),
                 lambda: opt.load(torch.zeros(40, device="cuda"), torch.zeros(40, device="cuda"), 1),
                 lambda: opt.load(torch.zeros(128, device="cuda"), torch.zeros(128, device="cuda"), -1)):
        with pytest.raises(GsxHipError):
            call()
    opt.groups[0]["beta1"] = 1.0
    with pytest.raises(GsxHipError):
        opt.step()
    assert opt.steps.item() == 0
