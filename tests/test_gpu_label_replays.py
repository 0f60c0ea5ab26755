"""Steps and answers of a label field captured into graphs: every replay is the step or the answer that an eager call would be, on
the head as it is by then, whichever of the two went before."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROWS, CODES, LABELS, FEATURES, TOP = 500, 40, 33, 70, 4


def data(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(-1, CODES, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
    labels = torch.randint(-1, LABELS, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
    weight = torch.rand(ROWS, device="cuda", generator=g) * (codes >= 0)
    ids = torch.stack([torch.randperm(LABELS, device="cuda", generator=g)[:TOP] for _ in range(ROWS)]).int()
    return codes, labels, weight, ids, torch.randn(ROWS, TOP, device="cuda", generator=g)


def capture(call):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = call()
    return graph, result


def state(field):
    return [field.table, field.head, field.table_grad, field.head_grad, *field.optimizer.moments(), field.blocks.values,
            field.blocks_t.values]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("given", [True, False])
def test_replayed_steps_go_on_from_the_last_one(bits, given):
    """Replays and eager steps in turn, each on new rows, beside a twin whose steps are all eager: the same bits."""
    from gsx_amd.label_field import LabelField
    field, twin = (LabelField(CODES, FEATURES, LABELS, moments=bits, weight_decay=0.01) for _ in range(2))
    batch = data(1)

    def step(f, b):
        codes, labels, weight, ids, logits = b
        return f.step_labels(codes, labels, weight, 0.125) if given else f.step(codes, ids, logits, weight)

    graph, loss = capture(lambda: step(field, batch))
    assert all(torch.equal(a, b) for a, b in zip(state(field), state(twin)))  # a capture computes nothing
    losses = []
    for k in range(6):
        for t, new in zip(batch, data(20 + k)):
            t.copy_(new)
        if k == 3:
            got = step(field, batch)
        else:
            graph.replay()
            got = loss
        want = step(twin, batch)
        torch.cuda.synchronize()
        assert torch.equal(got, want), k
        for a, b in zip(state(field), state(twin)):
            assert torch.equal(a, b), k
        losses.append(want.clone())
    assert field.optimizer.steps.item() == 6
    assert not torch.equal(losses[0], losses[1])


def test_replayed_steps_train():
    """The same rows again and again: the losses of replays fall as eager ones do, which those of a head that stays do not."""
    from gsx_amd.label_field import LabelField
    field, twin = (LabelField(CODES, FEATURES, LABELS, moments=32, learning_rate=0.05) for _ in range(2))
    codes, labels, weight, _, _ = data(3)
    graph, loss = capture(lambda: field.step_labels(codes, labels, weight))
    for _ in range(20):
        graph.replay()
        want = twin.step_labels(codes, labels, weight)
    assert torch.equal(loss, want)


@pytest.mark.parametrize("moments", [None, 32])
def test_replayed_logits_follow_eager_steps(moments):
    from gsx_amd.label_field import LabelField
    field = LabelField(CODES, FEATURES, LABELS, moments=moments)
    codes, labels, weight, ids, teacher = data(5)
    asked = codes[:9].clone()
    graph, logits = capture(lambda: field.logits(asked))
    for k in range(4):
        asked.copy_(codes[9 * k: 9 * k + 9])
        graph.replay()
        want = field.logits(asked)
        torch.cuda.synchronize()
        assert torch.equal(logits, want)
        field.step(codes, ids, teacher, weight)
        torch.cuda.synchronize()


def test_a_captured_step_with_adam_is_refused():
    """Adam's count of steps is the host's: a replay cannot go on with it."""
    from gsx_amd._lib import GsxHipError
    from gsx_amd.label_field import LabelField
    field = LabelField(CODES, FEATURES, LABELS)
    codes, labels, weight, ids, logits = data(7)

    def refused():
        for call in (lambda: field.step_labels(codes, labels, weight), lambda: field.step(codes, ids, logits, weight)):
            with pytest.raises(GsxHipError, match="AdamW"):
                call()
        return codes.clone()

    before = [t.clone() for t in (field.table, field.head)]
    graph, copy = capture(refused)
    graph.replay()
    assert torch.equal(copy, codes)
    assert all(torch.equal(a, b) for a, b in zip(before, (field.table, field.head)))
    assert all(g["step"] == 0 for g in field.optimizer.groups)
    assert torch.isfinite(field.step_labels(codes, labels, weight)).all()


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (33, 70), (70, 130), (5, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_into_blocks(rows, cols, dtype, transpose):
    """What is written is what a call of its own would give, within the blocks' rows alone, and where they were."""
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    want = fields.quantize(x, transpose)
    n, k = want.rows, want.cols
    wide, words = want.values.shape[1], want.exponents.shape[1]
    blocks = -(-k // 128)
    room = torch.full((n + 2, wide + 32), 7, dtype=torch.uint8, device="cuda")
    exponents = torch.full((n + 2, words + 8), 9, dtype=torch.uint8, device="cuda")
    out = fields.Blocks(room[1: n + 1, 16: 16 + wide], exponents[1: n + 1, 4: 4 + words], k)
    got = fields.quantize(x, transpose, out=out)
    assert got is out
    assert torch.equal(out.values, want.values) and torch.equal(out.exponents[:, :blocks], want.exponents[:, :blocks])
    assert torch.equal(got.float(), want.float())
    out.values.fill_(7)
    out.exponents.fill_(9)
    assert (room == 7).all() and (exponents == 9).all()


def same_answers(got, want):
    return all(torch.equal(a, b) for a, b in zip(got[:5], want[:5]))


@pytest.mark.parametrize("asked_before", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_answers_follow_replayed_steps(bits, asked_before):
    """Eager answers, captured ones and the head's 4-bit blocks between replays of a step and eager steps, beside an eager twin."""
    from gsx_amd import fields
    from gsx_amd.label_field import LabelField
    field, twin = (LabelField(CODES, FEATURES, LABELS, moments=bits, learning_rate=0.05) for _ in range(2))
    codes, labels, weight, _, _ = data(9)
    if asked_before:
        assert same_answers(field.answers(codes, 5, labels), twin.answers(codes, 5, labels))
    graph, _ = capture(lambda: field.step_labels(codes, labels, weight))
    asking, captured = capture(lambda: field.answers(codes, 5, labels))
    seen = []
    for k in range(5):
        if k == 2:
            field.step_labels(codes, labels, weight)
        else:
            graph.replay()
        twin.step_labels(codes, labels, weight)
        want = twin.answers(codes, 5, labels)
        asking.replay()
        got = field.answers(codes, 5, labels)
        torch.cuda.synchronize()
        assert same_answers(got, want), k
        assert same_answers(captured, want), k
        assert torch.equal(field.head_blocks4().float(), fields.quantize4(field.head).float())
        seen.append(want.chosen.clone())
    assert not torch.equal(seen[0], seen[1])


def test_answers_on_several_streams_wait_for_the_blocks():
    """The first answer after a step lays the head's 4-bit blocks out behind long work of its stream; answers on other streams, asked
    for at once, read them no earlier."""
    from gsx_amd.label_field import LabelField
    field, twin = (LabelField(CODES, FEATURES, LABELS, moments=32, learning_rate=0.2) for _ in range(2))
    codes, labels, weight, _, _ = data(11)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for k in range(4):
        field.step_labels(codes, labels, weight)
        twin.step_labels(codes, labels, weight)
        want = twin.answers(codes, 5, labels)
        torch.cuda.synchronize()
        got = []
        for at in range(3):
            with torch.cuda.stream(streams[(at + k) % 3]):
                if at == 0:
                    torch.cuda._sleep(20_000_000)
                got.append(field.answers(codes, 5, labels))
        torch.cuda.synchronize()
        assert all(same_answers(a, want) for a in got), k


def test_answers_of_a_head_that_was_read_in():
    """A head written over before the first answer is the one that answers."""
    from gsx_amd.label_field import LabelField
    field, other = LabelField(CODES, FEATURES, LABELS, seed=1), LabelField(CODES, FEATURES, LABELS, seed=2)
    codes = data(13)[0]
    field.table.copy_(other.table)
    field.head.copy_(other.head)
    assert same_answers(field.answers(codes, 5), other.answers(codes, 5))


@pytest.mark.parametrize("rows,cols", [(1, 1), (33, 70), (70, 130), (5, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize4_into_blocks(rows, cols, dtype):
    from gsx_amd import fields
    from gsx_amd._lib import GsxHipError
    g = torch.Generator("cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    want = fields.quantize4(x)
    wide, words, blocks = want.values.shape[1], want.exponents.shape[1], -(-cols // 32)
    room = torch.full((rows + 2, wide + 32), 7, dtype=torch.uint8, device="cuda")
    exponents = torch.full((rows + 2, words + 8), 9, dtype=torch.uint8, device="cuda")
    out = fields.Blocks4(room[1: rows + 1, 16: 16 + wide], exponents[1: rows + 1, 4: 4 + words], cols)
    assert fields.quantize4(x, out=out) is out
    assert torch.equal(out.values, want.values) and torch.equal(out.exponents[:, :blocks], want.exponents[:, :blocks])
    assert torch.equal(out.float(), want.float())
    out.values.fill_(7)
    out.exponents.fill_(9)
    assert (room == 7).all() and (exponents == 9).all()
    for bad in (fields.Blocks4(want.values, want.exponents, cols + 1), want.values,
                fields.Blocks4(want.values[:, : wide - 16], want.exponents, cols)):
        with pytest.raises(GsxHipError):
            fields.quantize4(x, out=bad)
