"""Reply controls on the GPU against oracle/logits_ref.py.

Float32 results equal the oracle's float32 operations bit for bit (each is rounded on its own, and IEEE), so picks are
equal at ties; 16-bit results are their roundings.  Against 64 bits a value may be off by the roundings it went through:
the quotient or product, frequency * count, the sum with presence, the difference, the sum with the bias, 2^-24 each of
what they round, and the output's own."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import logits_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def int32(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def f32(values):
    return torch.tensor(np.asarray(values), dtype=torch.float32, device=DEV)


def make_case(rows, vocab, history, biased, masked, dtype, seed=0):
    rng = np.random.RandomState(seed + vocab)
    c = {"logits": torch.tensor(rng.randn(rows, vocab) * 3, device=DEV).to(TYPES[dtype]),
         "tokens": rng.randint(-2, vocab + 2, (rows, history)),
         "lengths": np.minimum(rng.randint(0, history + 1, rows), history)}
    c["lengths"][0] = history
    if history:
        c["tokens"][:, ::3] = rng.randint(0, min(vocab, 7), c["tokens"][:, ::3].shape)  # some of them often
    c["reply"] = (c["lengths"] * rng.rand(rows)).astype(int)
    c["repetition"] = rng.choice([1.0, 1.1, 0.8, 1.7], rows).astype(np.float32)
    c["presence"] = rng.choice([0.0, 0.3, -0.7], rows).astype(np.float32)
    c["frequency"] = rng.choice([0.0, 0.11, -0.2], rows).astype(np.float32)
    c["bias"] = [[(int(t), float(np.float32(v))) for t, v in zip(rng.randint(0, vocab, biased), rng.randn(biased) * 4)]
                 for _ in range(rows)] if biased else None
    c["allowed"] = rng.rand(rows, vocab) < rng.rand(rows, 1) if masked else None
    if masked:
        c["allowed"][-1] = False  # a row whose mask leaves nothing
        c["none"] = rng.rand(rows) < 0.3  # and rows without a mask
        c["none"][-1] = False
    return c


def controls_of(c):
    from reply_controls import ReplyControls, pack_allowed

    rows, vocab = c["logits"].shape
    bias = None
    if c["bias"]:
        bias = (int32(t for row in c["bias"] for t, _ in row), f32([v for row in c["bias"] for _, v in row]),
                int32(np.cumsum([0] + [len(row) for row in c["bias"]])))
    allowed = None
    if c["allowed"] is not None:
        allowed = (pack_allowed(torch.tensor(c["allowed"], device=DEV)), int32(np.where(c["none"], -1, np.arange(rows))))
    return ReplyControls(rows, vocab, f32(c["repetition"]), f32(c["presence"]), f32(c["frequency"]), bias, allowed, DEV)


def apply(c, controls=None, ids=torch.int64, **kwargs):
    controls = controls or controls_of(c)
    return controls.apply(c["logits"], torch.tensor(c["tokens"], dtype=ids, device=DEV), int32(c["lengths"]),
                          int32(c["reply"]), **kwargs)


def check(c, out, pick):
    for r in range(c["logits"].shape[0]):
        args = (c["logits"][r].float().cpu().numpy(), c["tokens"][r][:c["lengths"][r]].tolist(), c["reply"][r],
                c["repetition"][r], c["presence"][r], c["frequency"][r], c["bias"][r] if c["bias"] else (),
                c["allowed"][r] if c["allowed"] is not None and not c["none"][r] else None)
        single, want_pick = logits_ref.adjust(*args, dtype=np.float32)
        assert int(pick[r]) == want_pick, r
        want = torch.tensor(single).to(out.dtype)
        assert torch.equal(out[r].cpu(), want), r
        whole, _ = logits_ref.adjust(*args)
        with np.errstate(all="ignore"):
            off = np.abs(np.where(whole == single, 0.0, whole - out[r].double().cpu().numpy()))
        size = np.where(np.isfinite(whole), np.abs(whole), 0.0) + 32.0  # penalties and biases below 32 in sum
        assert (off <= STEP[out.dtype] * size + 5 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,history,biased,masked", [
    (1, 1, 1, 0, False), (1, 31, 5, 3, True), (3, 33, 40, 9, True), (2, 256, 0, 0, True), (5, 1000, 300, 0, False),
    (4, 4099, 64, 7, True), (3, 8192, 2000, 40, False), (2, 8200, 700, 300, True), (2, 20001, 5000, 5, True)])
def test_shapes(rows, vocab, history, biased, masked, dtype):
    print(f"[case] logits {rows}x{vocab} history={history} biased={biased} masked={masked} {dtype}", flush=True)
    c = make_case(rows, vocab, history, biased, masked, dtype)
    check(c, *apply(c))
    check(c, *apply(c, ids=torch.int32))


def test_large_vocabulary():
    c = make_case(2, 128256, 1500, 20, True, "bf16")
    check(c, *apply(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(dtype):
    """Enough rows for the long stretches, two lines or four a thread."""
    c = make_case(70, 128256, 400, 9, True, dtype)
    out, pick = apply(c)
    for r in (0, 1, 33, 68, 69):
        one = {k: (v[r:r + 1] if k != "bias" else [v[r]]) for k, v in c.items()}
        check(one, out[r:r + 1], pick[r:r + 1])


def test_long_history():
    """More mentions than 15 bits count: 40,000 tokens, 35,000 of them one."""
    c = make_case(2, 9000, 40000, 3, False, "f32")
    c["tokens"][0, 2000:37000] = 17
    c["reply"][:] = [1000, 39000]
    c["lengths"][:] = 40000
    check(c, *apply(c))
    check(c, *apply(c, ids=torch.int32))


def test_in_place_and_strided():
    """Logits changed in place, rows that lie apart and begin anywhere, a given out of another alignment."""
    c = make_case(4, 777, 50, 5, True, "bf16")
    plain = c["logits"].clone()
    wide = torch.zeros(4, 803, dtype=torch.bfloat16, device=DEV)
    for start in (0, 3, 8):
        c["logits"] = wide[:, start:start + 777]
        c["logits"].copy_(plain)
        check(c, *apply(c))
        other = torch.full((4, 790), 9.0, dtype=torch.bfloat16, device=DEV)
        out, pick = apply(c, out=other[:, 5:782])
        check(c, out, pick)
        assert (other[:, :5] == 9.0).all() and (other[:, 782:] == 9.0).all()
        view = wide[:, start:start + 777]
        out, pick = apply(c, out=view)
        assert out is view
        c["logits"] = plain
        check(c, out, pick)
        assert not wide[:, :start].any() and not wide[:, start + 777:].any()
        wide.zero_()
    c["logits"] = plain.t().contiguous().t()  # columns contiguous: copied
    check(c, *apply(c))


def test_infinities_and_nan():
    from reply_controls import ReplyControls

    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[1.0, nan, 3.0, 4.0], [-inf, -inf, -inf, -inf], [inf, 2.0, inf, nan], [-inf, -5.0, -inf, -5.0],
                           [0.0, -0.0, -1.0, -1.0]], device=DEV)
    mask = torch.tensor([[1, 0, 1, 1], [1, 1, 1, 1], [0, 1, 1, 0], [1, 1, 1, 1], [0, 1, 0, 0]], device=DEV).bool()
    out, pick = ReplyControls(5, 4).apply(logits)
    assert torch.equal(out.isnan(), logits.isnan()) and pick.tolist() == [1, -1, 3, 1, 0]
    out, pick = ReplyControls(5, 4, allowed=mask).apply(logits)
    assert pick.tolist() == [3, -1, 2, 1, 1]
    assert not out.isnan().any() and (out[~mask] == -inf).all() and torch.equal(out[mask], logits[mask])
    # infinities under penalties stay what arithmetic makes of them; +0 and -0 are a tie
    out, pick = ReplyControls(5, 4, repetition=2.0, presence=1.0, bias={0: -inf}).apply(
        logits, torch.arange(4, device=DEV).expand(5, 4))
    assert out[3].tolist() == [-inf, -11.0, -inf, -11.0] and pick[3] == 1
    assert out[2][:3].tolist()[1:] == [0.0, inf] and out[4].tolist() == [-inf, -1.0, -3.0, -3.0]
    assert torch.tensor([[0.0, -0.0], [-0.0, 0.0]], device=DEV).argmax(1).tolist() == \
        ReplyControls(2, 2).apply(torch.tensor([[0.0, -0.0], [-0.0, 0.0]], device=DEV))[1].tolist()


def test_masks_change_and_repeat():
    """The mask replaced between steps; one mask for every row; the same bias id three times: its last value counts."""
    from reply_controls import ReplyControls

    logits = torch.randn(3, 100, device=DEV)
    controls = ReplyControls(3, 100, bias=(int32([7, 7, 7, 50]), f32([1.0, 2.0, 300.0, -1.0]), int32([0, 3, 4, 4])))
    out, pick = controls.apply(logits)
    want = logits.clone()
    want[0, 7] += 300.0
    want[1, 50] -= 1.0
    assert torch.equal(out, want) and pick[0] == 7
    only = torch.zeros(1, 100, dtype=torch.bool, device=DEV)
    for token in (99, 31, 32, 0):
        only.zero_()
        only[0, token] = True
        controls.allow(only)
        assert controls.apply(logits)[1].tolist() == [token] * 3
    controls.allow(None)
    assert torch.equal(controls.apply(logits)[0], want)


def test_graph_and_stream():
    c = make_case(3, 5000, 200, 5, True, "f16")
    controls = controls_of(c)
    tokens, lengths, reply = torch.tensor(c["tokens"], device=DEV), int32(c["lengths"]), int32(c["reply"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check(c, *controls.apply(c["logits"], tokens, lengths, reply))
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, pick = controls.apply(c["logits"], tokens, lengths, reply)
    for turn in range(4):
        c["logits"].copy_(torch.randn(3, 5000, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out, pick)
        controls.apply(c["logits"])


@pytest.mark.parametrize("masks", [1, 3])
def test_masks_change_under_a_graph(masks):
    """Replays of a captured call see the bool masks given since, also with masks of another shape or none between."""
    from reply_controls import ReplyControls

    rows, vocab = 3, 1000
    generator = torch.Generator(DEV).manual_seed(4)
    logits = torch.randn(rows, vocab, generator=generator, device=DEV)
    mask = lambda n: torch.rand(n, vocab, generator=generator, device=DEV) < 0.1
    controls = ReplyControls(rows, vocab, allowed=mask(masks), device=DEV)
    controls.apply(logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, pick = controls.apply(logits)
    for turn in range(4):
        if turn == 2:
            controls.allow(None)
            controls.allow(mask(4 - masks))
        may = mask(masks)
        controls.allow(may.cpu() if turn == 1 else may)
        torch.full((1 << 16,), -1, dtype=torch.int32, device=DEV)  # what memory given back would hold
        graph.replay()
        want = torch.where(may, logits, -float("inf")).argmax(1)
        assert torch.equal(pick, want) and torch.equal(controls.apply(logits)[1], want)


@pytest.mark.parametrize("rows,dtype,vocabs", [(2, "f16", (8185, 8186, 8191, 16383)), (2, "bf16", (8186, 8191, 32767)),
                                               (2, "f32", (4093, 4094, 4095, 8191)), (64, "bf16", (131070, 131071)),
                                               (64, "f32", (131070, 131071))])
def test_vocabularies_below_a_stretch(rows, dtype, vocabs):
    """The last stretch of a row begins past the vocabulary: it counts nothing, and the others count as ever."""
    for vocab in vocabs:
        print(f"[case] logits {rows}x{vocab} {dtype}", flush=True)
        c = make_case(rows, vocab, 500, 6, True, dtype)
        out, pick = apply(c)
        for r in (0, 1, rows - 1):
            one = {k: (v[r:r + 1] if k != "bias" else [v[r]]) for k, v in c.items()}
            check(one, out[r:r + 1], pick[r:r + 1])


@pytest.mark.parametrize("vocab,biases", [(300, 0), (300, 3), (9000, 2)])
def test_mask_numbers_past_the_masks(vocab, biases):
    """A row whose mask number is past the masks may take nothing; one below 0 has no mask."""
    from reply_controls import ReplyControls, pack_allowed

    logits = torch.randn(5, vocab, device=DEV)
    mask = torch.rand(2, vocab, device=DEV) < 0.5
    controls = ReplyControls(5, vocab, bias={t * 7: 1.0 for t in range(biases)} or None,
                             allowed=(pack_allowed(mask), int32([0, 2, -1, 2**31 - 1, -(2**31)])))
    out, pick = controls.apply(logits, torch.arange(50, device=DEV).expand(5, 50))
    free, best = ReplyControls(5, vocab, bias={t * 7: 1.0 for t in range(biases)} or None).apply(
        logits, torch.arange(50, device=DEV).expand(5, 50))
    assert (out[[1, 3]] == -float("inf")).all() and pick[[1, 3]].tolist() == [-1, -1]
    assert torch.equal(out[[2, 4]], free[[2, 4]]) and torch.equal(pick[[2, 4]], best[[2, 4]])
    assert torch.equal(out[0], torch.where(mask[0], free[0], -float("inf")))


@pytest.mark.parametrize("masks", [1, 2])
def test_a_copy_keeps_its_masks(masks):
    """Bool masks given to controls after they were copied, or to the copy, are theirs alone."""
    import copy

    from reply_controls import ReplyControls

    only = lambda token: (torch.arange(100, device=DEV) == token).expand(masks, 100)
    logits = torch.randn(2, 100, device=DEV)
    controls = ReplyControls(2, 100, allowed=only(7))
    other = copy.copy(controls)
    controls.allow(only(9))
    assert other.apply(logits)[1].tolist() == [7, 7] and controls.apply(logits)[1].tolist() == [9, 9]
    other.allow(only(11))
    third = copy.copy(other)
    other.allow(None)
    assert controls.apply(logits)[1].tolist() == [9, 9] and third.apply(logits)[1].tolist() == [11, 11]
    assert torch.equal(other.apply(logits)[1], logits.argmax(1))


def test_bias_lists_are_fixed():
    """Ids and rows of a tuple of biases changed later have no part (rows could come to hold an id twice); values have."""
    from reply_controls import ReplyControls

    logits = torch.randn(2, 100, device=DEV)
    ids, values, cu = int32([7, 8, 7, 50]), f32([1.0, 2.0, 4.0, 8.0]), int32([0, 2, 4])
    controls = ReplyControls(2, 100, bias=(ids, values, cu))
    ids.fill_(3)
    cu.copy_(int32([0, 4, 4]))
    want = logits.clone()
    want[0, 7], want[0, 8], want[1, 7], want[1, 50] = want[0, 7] + 1, want[0, 8] + 2, want[1, 7] + 4, want[1, 50] + 8
    assert torch.equal(controls.apply(logits)[0], want)
    values.mul_(2.0)
    out = controls.apply(logits)[0]
    assert torch.equal(out[0, 7], logits[0, 7] + 2.0) and torch.equal(out[1, 50], logits[1, 50] + 16.0)


def test_results_over_other_logits_are_refused():
    """A result may lie in its logits' place, or between their rows, but not over others'."""
    from reply_controls import ReplyControls

    wide = torch.randn(5, 700, device=DEV)
    controls, given = ReplyControls(4, 300, repetition=2.0), wide.clone()
    history = torch.arange(40, device=DEV).expand(4, 40)
    want, _ = controls.apply(given[:4, :300], history)
    for out in (wide[1:, :300], wide[:4, 1:301], wide.view(-1)[:1200].view(4, 300), wide[:4, 299:599]):
        with pytest.raises(ValueError, match="other logits"):
            controls.apply(wide[:4, :300], history, out=out)
    assert torch.equal(wide, given)
    for out in (wide[:4, 300:600], wide[1:, 301:601], wide[:4, :300]):
        assert torch.equal(controls.apply(wide[:4, :300], history, out=out)[0], want)


@pytest.mark.parametrize("given", ["nothing", "a result", "the logits' place"])
def test_recorded_calls_have_no_gradient(given):
    from reply_controls import ReplyControls

    logits = torch.randn(3, 400, device=DEV)
    controls = ReplyControls(3, 400, bias={5: 1.0})
    want, best = controls.apply(logits)
    assert not want.requires_grad
    rows = logits.clone().requires_grad_() * 1.0
    out = {"nothing": None, "a result": torch.empty_like(logits), "the logits' place": rows}[given]
    got, pick = controls.apply(rows, out=out)
    assert got.requires_grad and torch.equal(got, want) and torch.equal(pick, best) and (out is None or got is out)
    with pytest.raises(RuntimeError, match="no backward pass"):
        got.sum().backward()
    assert not controls.apply(rows.detach())[0].requires_grad


def test_a_recorded_leaf_is_not_written():
    from reply_controls import ReplyControls

    leaf = torch.randn(3, 400, device=DEV).requires_grad_()
    given = leaf.detach().clone()
    for place in (leaf, leaf[:]):
        with pytest.raises(RuntimeError, match="leaf"):
            ReplyControls(3, 400, bias={5: 1.0}).apply(leaf, out=place)
    assert torch.equal(leaf, given)
