"""Batched decoding over a paged cache: the graph operator, the page bookkeeping, ``PagedDecoder`` and token rules.

CPU: the operator's plain form against 64 bits, its lowering, ``PagedDecoder`` over a byte-addressed stand-in for device
memory computing with the eager module. GPU (marked): compiled operators and whole models against the same."""

from __future__ import annotations

import ctypes
import math
from pathlib import Path

import numpy as np
import pytest
import torch

import chroma_amd
from chroma_amd import Decoder, PagedDecoder, Program, TokenRules
from chroma_amd._src import native
from chroma_amd._src.build import build
from chroma_amd._src.codegen.hip import HIPCodegen
from chroma_amd._src.compiler import lower_program
from chroma_amd._src.decoder import _select_host
from chroma_amd._src.dtypes import BFLOAT16, bf16_to_float32, float32_to_bf16
from chroma_amd._src.paged import PagePool
from chroma_amd._src.rules import pack
from chroma_amd.models.cached import export_cached
from chroma_amd.models.paged import export_paged
from chroma_amd.ops import paged_attention
from oracle import compile_cpu
from tests.helpers import Function, as_float, numpy_of, random_transformer, small_config
from tests.test_batched_operators import adjust_reference, attention_reference, paged_inputs
from tests.test_decoder import FakeDevice, FakeDeviceProgram, FakeNative

gpu = pytest.mark.gpu
IDS = dict(ids=["f32", "bf16"])


# ------------------------------------------------------------------------------------------------ the operator
def operator_arguments(inputs):
    return [inputs[name] for name in ("q", "k_pages", "v_pages", "k_new", "v_new", "table", "lengths", "sinks")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], **IDS)
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("window,first", [(0, 0), (5, 0), (7, 3)])
def test_plain_form_of_the_operator(window, first, fresh, dtype):
    inputs = paged_inputs([0, 1, 20, 33], kv=2, group=3, dim=16, page=8, dtype=dtype, fresh=fresh, sinks=window == 0, seed=window)
    inputs["table"][2, 1] = len(inputs["k_pages"])
    inputs["lengths"][1] = -4
    want, bound = attention_reference(**inputs, window=window, first=first)
    got = paged_attention(*operator_arguments(inputs), 0.25, window, first).double()
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all()


def test_operator_refusals():
    good = operator_arguments(paged_inputs([5, 9], kv=2, group=2, dim=8, page=4, dtype=torch.float32))
    paged_attention(*good, 1.0)
    for index, value, kind in ((0, good[0][0], ValueError), (1, good[1][:, :, :1], ValueError), (3, None, ValueError), (3, good[3][:1], ValueError),
                               (0, good[0][:0], ValueError), (5, good[5].int(), TypeError), (5, good[5][:1], ValueError), (6, good[6][:1], ValueError), (7, good[7][:3], ValueError),
                               (2, good[2].bfloat16(), TypeError), (7, good[7].double(), TypeError)):
        changed = list(good)
        changed[index] = value
        with pytest.raises(kind):
            paged_attention(*changed, 1.0)
    for window, first in ((-1, 0), (0, -1)):
        with pytest.raises(ValueError):
            paged_attention(*good, 1.0, window, first)
    for empty in (good[1][:0], good[1][:, :0]):
        with pytest.raises(ValueError, match="empty"):
            paged_attention(good[0], empty, empty, *good[3:], 1.0)


class Attention(torch.nn.Module):
    """The operator on one layer of a cache; q and the new rows are expressions or views, as in a model."""

    def __init__(self, layer, window, first, scale, off=0):
        super().__init__()
        self.layer, self.window, self.first, self.scale, self.off = layer, window, first, scale, off

    def forward(self, q, k_pages, v_pages, k_new, v_new, table, lengths, sinks):
        pages = k_pages.shape[1:]
        k, v = (x[self.layer : self.layer + 1].reshape(pages) for x in (k_pages, v_pages))
        if self.off:  # operands that start off 16 bytes
            flat = q.shape[0] * q.shape[1] * q.shape[2] * q.shape[3]
            q = torch.cat((q.reshape(-1)[:1], q.reshape(-1))).contiguous()[1 : 1 + flat].reshape(q.shape)
        return paged_attention(q * 1.0 if not self.off else q, k, v, k_new, v_new, table, lengths, sinks, self.scale, self.window, self.first)


def exported(inputs, *, window=0, first=0, off=0):
    """(exported module, its arguments): the pages as layer 1 of 2."""
    arguments = operator_arguments(inputs)
    for i in (1, 2):
        arguments[i] = torch.stack((torch.zeros_like(arguments[i]), arguments[i]))
    module = Attention(1, window, first, inputs["q"].shape[-1] ** -0.5, off)
    present = [x for x in arguments if x is not None]
    holes = [x is None for x in arguments]

    def call(*given):
        rest = iter(given)
        return module(*(None if hole else next(rest) for hole in holes))

    return torch.export.export(Function(call), tuple(present)), present


@pytest.mark.parametrize("lengths,window,kernels", [([40, 3], 0, ["whole"]), ([4000, 3], 0, ["shares", "combine"]), ([4000, 3], 100, ["whole"])])
def test_lowering_cuts_by_the_span_and_the_window(tmp_path, lengths, window, kernels):
    graph, _ = exported(paged_inputs(lengths, kv=2, group=4, dim=64, page=16, dtype=torch.bfloat16), window=window)
    generated = lower_program(graph, HIPCodegen())
    source = generated.files["model.hip"]
    assert [name for name in ("whole", "shares", "combine") if f"attention_paged_{name}<" in source] == kernels
    assert generated.stats["fused_attentions"] == 1
    build(generated, tmp_path, load=False)  # hipcc accepts it


def test_lowering_refusals():
    for dim, message in ((12, "heads of 12"), (264, "heads of 264")):
        graph, _ = exported(paged_inputs([5], kv=1, group=1, dim=dim, page=4, dtype=torch.float32))
        with pytest.raises(NotImplementedError, match=message):
            lower_program(graph, HIPCodegen())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], **IDS)
@pytest.mark.parametrize("lengths,shape,fresh,window,first,off", [
    ([40, 3, 0], (2, 4, 16, 8), True, 0, 0, 0), ([40, 3, 0], (2, 4, 16, 8), False, 0, 0, 1), ([700, 3000, 1], (2, 8, 64, 16), True, 0, 0, 0),
    ([700, 3000, 1], (1, 3, 80, 16), False, 200, 5, 1), ([3000, 10], (1, 20, 32, 64), True, 1800, 70, 0)])
def test_compiled_operator(tmp_path, lengths, shape, fresh, window, first, off, dtype):
    kv, group, dim, page = shape
    inputs = paged_inputs(lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=fresh, sinks=fresh, seed=dim)
    want, bound = attention_reference(**inputs, window=window, first=first)
    graph, arguments = exported(inputs, window=window, first=first, off=off)
    with chroma_amd.compile(graph, tmp_path) as program:
        for _ in range(3):  # graph replays
            got = torch.from_numpy(as_float(program(*arguments)).copy()).double()
            assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all()


# ------------------------------------------------------------------------------------------------ pages
def test_page_pool_against_a_plain_count():
    """Random takes, shares, releases and compactions: references, free pages and where the live ones lie."""
    rng = np.random.default_rng(3)
    pool, owners = PagePool(12), []
    for _ in range(400):
        action = rng.integers(4)
        if action == 0 and pool.free:
            lowest = min(set(range(12)) - {page for owner in owners for page in owner})
            owners.append([pool.take()])
            assert owners[-1] == [lowest]
        elif action == 1 and owners:
            owners.append(list(owners[rng.integers(len(owners))]))
            pool.share(owners[-1])
        elif action == 2 and owners:
            pool.release(owners.pop(rng.integers(len(owners))))
        elif action == 3:
            moves = pool.compaction()
            live = {page for owner in owners for page in owner}
            assert not set(moves) - live and not set(moves.values()) & live and len(set(moves.values())) == len(moves)
            pool.move(moves)
            owners = [[moves.get(page, page) for page in owner] for owner in owners]
            assert {page for owner in owners for page in owner} == set(range(len(live)))
        counts = np.bincount([page for owner in owners for page in owner], minlength=12)
        np.testing.assert_array_equal(pool.references, counts)
        assert pool.free == int((counts == 0).sum())
    while pool.free:
        pool.take()
    with pytest.raises(RuntimeError, match="no free page"):
        pool.take()


# ------------------------------------------------------------------------------------------------ the decoder
class EagerProgram:
    """What ``FakeNative`` computes with: the eager module of an export, called with arrays."""

    def __init__(self, graph) -> None:
        self.module = graph.module()
        names = {torch.float32: "float32", torch.int64: "int64"}
        nodes = {node.name: node.meta["val"] for node in graph.graph.nodes if "val" in node.meta}
        self.inputs, self.outputs = ([{"name": name, "shape": list(nodes[name].shape), "dtype": names[nodes[name].dtype]} for name in chosen]
                                     for chosen in (graph.graph_signature.user_inputs, graph.graph_signature.user_outputs))
        self.stats = {}

    def __call__(self, *arrays):
        if (arrays[0] < 0).any() or (arrays[0] >= 17).any():
            raise IndexError("Tensor index out of range")
        with torch.no_grad():
            return [value.numpy() for value in self.module(*(torch.from_numpy(a.copy()) for a in arrays))]


class FakePagedNative(FakeNative):
    def clear_input(self, index):
        self.device.view(self.inputs[index], self.oracle.inputs[index])[...] = 0

    def cache_move(self, to, source, layers, row_bytes, moves):
        moves = np.array(moves).reshape(-1, 3)

        def move():
            memory = self.device.memory
            for which in ("keys", "values"):
                taken = []
                for first, _, rows in moves:
                    assert 0 <= first and first + rows <= source.rows
                    taken.append([memory[getattr(source, which) + n * source.layer_pitch + first * row_bytes :][: rows * row_bytes].copy()
                                  for n in range(layers)])
                for (_, first, rows), data in zip(moves, taken):
                    assert 0 <= first and first + rows <= to.rows
                    for n in range(layers):
                        memory[getattr(to, which) + n * to.layer_pitch + first * row_bytes :][: rows * row_bytes] = data[n]

        self.pending.append(move)

    def run_top(self, inputs, outputs, index, k, rules=None):
        spec = self.oracle.outputs[index]
        self.run(inputs, outputs, resident=True)
        rows = self.device.view(self.outputs[index], spec)
        chosen = [_select_host((rules[i] if rules else TokenRules()).apply(row), k, None) for i, row in enumerate(rows)]
        return np.stack([values for values, _ in chosen]), np.stack([ids for _, ids in chosen])


class FakePagedProgram(FakeDeviceProgram):
    def __init__(self, graph, device) -> None:
        super().__init__(EagerProgram(graph), device)
        self._model = FakePagedNative(EagerProgram(graph), device)

    def close(self):
        pass


CONTEXT, SLOTS, PAGES, ROWS, SPAN = 9, 4, 14, 3, 5


def small_model(head_dim=8, **changes):
    return random_transformer(small_config(num_hidden_layers=2, head_dim=head_dim, hidden_size=16, num_attention_heads=4, num_key_value_heads=2,
                                           sliding_window=4, **changes), seed=5, std=0.2)


def fake_paged_decoder(model, pages=PAGES):
    device = FakeDevice(1 << 22)
    prompts = [FakePagedProgram(export_cached(model, CONTEXT, steps), device) for steps in (CONTEXT, 1)]
    return PagedDecoder(Decoder(*prompts, sliding_window=4), FakePagedProgram(export_paged(model, SLOTS, pages, ROWS, SPAN), device))


class Twin:
    """The texts of a ``PagedDecoder``'s sequences, and the eager model's logits after each."""

    def __init__(self, model, rtol, atol) -> None:
        self.model, self.texts, self.tolerance = model, {}, dict(rtol=rtol, atol=atol)

    def check(self, sequence, logits):
        with torch.no_grad():
            want = self.model(torch.tensor(self.texts[sequence]))[-1]
        np.testing.assert_allclose(as_float(logits), want.float().numpy(), **self.tolerance)

    def step(self, decoder, tokens):
        logits = decoder.step(tokens)
        for (sequence, token), row in zip(tokens.items(), logits):
            self.texts[sequence].append(token)
            self.check(sequence, row)
            assert decoder.position(sequence) == len(self.texts[sequence])


def live_pages(decoder):
    return {page for sequence in decoder.sequences for page in decoder.pages(sequence)}


def walk(decoder, twin, vocabulary):
    """A run as a program makes it: prompts, steps of some or all sequences, forks before and inside a page, ends, compaction."""

    def add(prompt):
        sequence, logits = decoder.add(prompt)
        twin.texts[sequence] = list(prompt)
        twin.check(sequence, logits[0])
        return sequence

    a, b = add([3, 1, 4, 1, 5]), add([9, 2, 6])
    twin.step(decoder, {a: 5, b: 3})
    twin.step(decoder, {b: 7})
    c = decoder.fork(a)  # a holds 6 rows: both begin a page of their own
    twin.texts[c] = list(twin.texts[a])
    twin.step(decoder, {c: 2, a: 8})
    assert decoder.pages(a)[:2] == decoder.pages(c)[:2] and decoder.pages(a)[2] != decoder.pages(c)[2]
    d = decoder.fork(b)  # b holds 5 rows: its second page is shared until one of them writes
    twin.texts[d] = list(twin.texts[b])
    assert decoder.pages(d) == decoder.pages(b)
    twin.step(decoder, {d: 11, b: 12, a: 1})
    assert decoder.pages(d)[0] == decoder.pages(b)[0] and decoder.pages(d)[1] != decoder.pages(b)[1]
    with pytest.raises(RuntimeError, match="holds 4 sequences"):
        decoder.fork(a)
    with pytest.raises(RuntimeError, match="holds 4 sequences"):
        decoder.add([1])
    decoder.free(a)
    before = live_pages(decoder)
    assert decoder.free_pages == PAGES - len(before)
    moved = decoder.compact()
    assert moved == len([page for page in before if page >= len(before)]) and live_pages(decoder) == set(range(len(before)))
    assert decoder.compact() == 0
    twin.step(decoder, {b: 4, c: 4, d: 4})
    e = add([7, 7, 7, 7, 7, 7, 7, 7])
    for token in (1, 2, 3):
        twin.step(decoder, {e: token, c: token + 1})
    for sequence in (b, c, d):
        decoder.free(sequence)
    twin.step(decoder, {e: 16})
    return e


def test_paged_decoder_matches_the_model_on_the_host():
    model = small_model()
    with fake_paged_decoder(model) as decoder:
        e = walk(decoder, Twin(model, 2e-5, 2e-6), 17)
        assert decoder.free_pages == PAGES - 4 and decoder.page_rows == ROWS
        while decoder.position(e) < SPAN * ROWS:
            decoder.step({e: 1})
        with pytest.raises(ValueError, match="all that the step program has pages for"):
            decoder.step({e: 1})


def test_paged_decoder_refuses_and_keeps_its_state():
    model = small_model()
    decoder = fake_paged_decoder(model, pages=11)
    twin = Twin(model, 2e-5, 2e-6)
    a, _ = decoder.add([1, 2, 3, 4, 5, 6])
    twin.texts[a] = [1, 2, 3, 4, 5, 6]
    state = (decoder.pages(a), decoder.position(a), decoder.free_pages)
    for tokens, kind in (({}, ValueError), ({a + 1: 1}, KeyError), ({a: 1.5}, TypeError), ({a: 17}, IndexError), ({a: -1}, IndexError)):
        with pytest.raises(kind):
            decoder.step(tokens)
        assert (decoder.pages(a), decoder.position(a), decoder.free_pages) == state
    for prompt, kind in (([], ValueError), (list(range(10)), ValueError), ([17], IndexError), ([0.5], TypeError)):
        with pytest.raises(kind):
            decoder.add(prompt)
        assert decoder.sequences == [a] and decoder.free_pages == state[2]
    for k in (0, 18, 2.0):
        with pytest.raises(ValueError):
            decoder.step_top({a: 1}, k)
    with pytest.raises(KeyError):
        decoder.step_top({a: 1}, rules={a + 1: TokenRules()})
    # three more sequences of 9 rows take the 9 pages left: a step in which all begin a page is refused whole
    others = [decoder.add([1] * 9)[0] for _ in range(3)]
    assert decoder.free_pages == 0
    with pytest.raises(RuntimeError, match="needs 4 pages, 0 are free"):
        decoder.step({a: 1, **{other: 1 for other in others}})
    assert decoder.position(a) == 6 and decoder.position(others[0]) == 9
    decoder.free(others[2])
    twin.step(decoder, {a: 2})
    with pytest.raises(RuntimeError, match="needs 3 pages, 2 are free"):
        decoder.add([1] * 9)

    def interrupted(inputs, outputs, *, resident):
        raise KeyboardInterrupt

    native_run, decoder._step.native.run = decoder._step.native.run, interrupted
    with pytest.raises(KeyboardInterrupt):
        decoder.step({a: 3})
    decoder._step.native.run = native_run
    twin.step(decoder, {a: 3})
    decoder.close()
    for call in (lambda: decoder.step({a: 1}), lambda: decoder.add([1]), lambda: decoder.fork(a), lambda: decoder.compact(), lambda: decoder.free(a)):
        with pytest.raises(RuntimeError, match="closed"):
            call()


def test_paged_decoder_refuses_programs_that_do_not_belong_together():
    model, other = small_model(), small_model(head_dim=16)
    device = FakeDevice(1 << 22)
    prompts = Decoder(*[FakePagedProgram(export_cached(model, CONTEXT, steps), device) for steps in (CONTEXT, 1)])
    for graph in (export_paged(other, SLOTS, PAGES, ROWS, SPAN), export_cached(model, CONTEXT, 1)):
        with pytest.raises(ValueError, match="PagedDecoder"):
            PagedDecoder(prompts, FakePagedProgram(graph, device))
    for part, index, shape in (("inputs", 3, [2, PAGES - 1, ROWS, 2, 8]), ("inputs", 5, [SLOTS + 1]), ("outputs", 1, [2, SLOTS - 1, 2, 8]),
                               ("outputs", 2, [1, SLOTS, 2, 8]), ("inputs", 0, [SLOTS + 1])):
        step = FakePagedProgram(export_paged(model, SLOTS, PAGES, ROWS, SPAN), device)
        getattr(step, part)[index]["shape"] = shape
        with pytest.raises(ValueError, match="same model"):
            PagedDecoder(prompts, step)
    for extents in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            export_paged(model, *extents)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], **IDS)
def test_paged_decoder_matches_the_model(tmp_path, dtype):
    model = small_model().to(dtype)
    prompts = [chroma_amd.compile(export_cached(model, CONTEXT, steps), tmp_path / f"p{steps}") for steps in (CONTEXT, 1)]
    step = chroma_amd.compile(export_paged(model, SLOTS, PAGES, ROWS, SPAN), tmp_path / "step")
    # bfloat16: the framework's tolerance for small whole models
    tolerance = (2e-5, 2e-6) if dtype == torch.float32 else (0.03, 0.03)
    with PagedDecoder(Decoder(*prompts, sliding_window=4), step) as decoder:
        walk(decoder, Twin(model, *tolerance), 17)


@gpu
def test_paged_decoder_of_long_texts(tmp_path):
    """Steps past the one-launch attention's rows: 2600 rows in pages of 32, the prompt in one call, two branches."""
    model = random_transformer(small_config(num_hidden_layers=2, head_dim=16, hidden_size=32, num_attention_heads=8, num_key_value_heads=2,
                                            sliding_window=50), seed=5, std=0.2)
    context = 2600
    prompts = [chroma_amd.compile(export_cached(model, context, steps), tmp_path / f"p{steps}") for steps in (context, 1)]
    step = chroma_amd.compile(export_paged(model, 3, 200, 32, 90), tmp_path / "step")
    text = (np.arange(context) * 7 % 17).tolist()
    twin = Twin(model, 1e-4, 1e-5)
    with PagedDecoder(Decoder(*prompts, sliding_window=50), step) as decoder:
        a, logits = decoder.add(text)
        twin.texts[a] = list(text)
        twin.check(a, logits[0])
        b = decoder.fork(a)
        twin.texts[b] = list(text)
        twin.step(decoder, {a: 3, b: 4})
        twin.step(decoder, {b: 5, a: 1})


# ------------------------------------------------------------------------------------------------ rules
def random_rules(rng, vocabulary, rows):
    """Rules of several rows, with and without each part."""
    rules = []
    for i in range(rows):
        bias = (None, {int(t): float(rng.normal()) for t in rng.integers(0, vocabulary, 5)}, rng.normal(size=vocabulary).astype(np.float32))[i % 3]
        allowed = (None, rng.integers(0, vocabulary, vocabulary // 2 + 1), rng.random(vocabulary) < 0.5)[(i // 2) % 3]
        rules.append(TokenRules(rng.integers(0, vocabulary, rng.integers(0, 20)), 0.5 + rng.random(), rng.normal(), rng.normal(), bias, allowed))
    return rules


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], **IDS)
def test_rules_on_the_host(dtype):
    """``apply`` and ``pack`` against the 64-bit rule."""
    rng, vocabulary = np.random.default_rng(1), 45
    rules = random_rules(rng, vocabulary, 12)
    logits = torch.from_numpy(rng.normal(size=(12, vocabulary)).astype(np.float32) * 4).to(dtype)
    arrays = {name: None if a is None else torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a) for name, a in pack(rules, vocabulary).items()}
    want, bound = adjust_reference(logits, lengths=arrays.pop("history_lengths"), **arrays)
    for row, rule, expected, limit in zip(numpy_of(logits), rules, want, bound):
        got = torch.from_numpy(as_float(rule.apply(row)).copy()).double()
        fine = torch.isfinite(expected)
        assert torch.equal(got[~fine], expected[~fine]) and ((got - expected).abs()[fine] <= limit[fine]).all()


def test_packed_rules_share_rows():
    bias, allowed = np.ones(40, np.float32), np.arange(40) % 2 == 0
    arrays = pack([TokenRules(bias=bias, allowed=allowed), TokenRules(bias=bias, allowed=allowed)], 40)
    # TokenRules keeps the arrays it is given, so equal ones are laid out once
    assert arrays["history"] is None and arrays["repetition"] is None
    assert arrays["bias"].shape == (1, 40) and arrays["mask"].tolist() == [[0x55555555, 0x55]]
    arrays = pack([TokenRules(history=[3], bias={2: 1.5}), TokenRules()], 40)
    assert arrays["history"].tolist() == [[3], [-1]] and arrays["history_lengths"].tolist() == [1, 0]
    assert arrays["bias"].shape == (2, 40) and arrays["bias"][0, 2] == 1.5 and not arrays["bias"][1].any() and arrays["mask"] is None


@pytest.mark.parametrize("arguments,kind", [
    (dict(repetition=0.0), ValueError), (dict(repetition=-1.0), ValueError), (dict(repetition=math.inf), ValueError), (dict(presence=math.nan), ValueError),
    (dict(frequency=math.inf), ValueError), (dict(history=[1.5]), TypeError), (dict(history=[[1]]), TypeError), (dict(bias=np.zeros((2, 2))), ValueError),
    (dict(allowed=[0.5]), TypeError), (dict(allowed=np.zeros((2, 2), bool)), TypeError),
    (dict(repetition=1e-60), ValueError), (dict(frequency=-1e39), ValueError)])
def test_rules_refuse(arguments, kind):
    with pytest.raises(kind):
        TokenRules(**arguments)


@pytest.mark.parametrize("arguments,kind", [(dict(history=[10]), IndexError), (dict(history=[-1]), IndexError), (dict(bias={10: 1.0}), IndexError),
                                            (dict(bias=np.zeros(9)), ValueError), (dict(allowed=[10]), IndexError), (dict(allowed=np.ones(11, bool)), ValueError),
                                            (dict(allowed=[]), ValueError), (dict(allowed=np.zeros(10, bool)), ValueError)])
def test_rules_refuse_another_vocabulary(arguments, kind):
    rules = TokenRules(**arguments)
    with pytest.raises(kind):
        rules.check(10)
    with pytest.raises(kind):
        rules.apply(np.zeros(10, np.float32))


def test_decoder_applies_rules_on_the_host(tmp_path):
    model = small_model()
    programs = [compile_cpu(export_cached(model, CONTEXT, steps), tmp_path / str(steps)) for steps in (CONTEXT, 1)]
    choosing, full = Decoder(*programs, sliding_window=4), Decoder(*programs, sliding_window=4)
    rules = random_rules(np.random.default_rng(2), 17, 6)
    for token, rule in zip((3, 1, 4, 1, 5, 9), rules):
        values, ids = choosing.append_top([token], 4, rules=rule)
        want_values, want_ids = _select_host(rule.apply(full.append([token])[0]), 4, None)
        np.testing.assert_array_equal(ids, want_ids)
        np.testing.assert_array_equal(values, want_values)
    only = TokenRules(allowed=[11])
    assert choosing.greedy([2], rules=only) == 11
    with pytest.raises(ValueError, match="rules"):
        choosing.append_top([1], 1, allowed=[3], rules=only)
    with pytest.raises(IndexError):
        choosing.append_top([1], 1, rules=TokenRules(history=[17]))
    assert choosing.position == 7


def test_paged_decoder_applies_rules_on_the_host():
    model = small_model()
    decoder = fake_paged_decoder(model)
    a, b = decoder.add([1, 2, 3])[0], decoder.add([4])[0]
    values, ids = decoder.step_top({b: 5, a: 6}, 3, rules={a: TokenRules(allowed=[13, 2]), b: TokenRules(history=[5, 5], presence=100.0)})
    assert set(ids[1][:2]) == {13, 2} and values[1][2] == -np.inf and 5 not in ids[0]
    values, ids = decoder.step_top({a: 7})
    assert ids.shape == values.shape == (1, 1)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], **IDS)
def test_rules_on_the_device(tmp_path, dtype):
    """``append_top`` and ``step_top`` with rules against the host rule on the logits that a twin downloads: values and ids
    bit for bit (the same float operations)."""
    model = small_model(vocab_size=3001).to(dtype)
    paths = [tmp_path / name for name in ("prefill", "one", "step")]
    for path, graph in zip(paths, (export_cached(model, CONTEXT, CONTEXT), export_cached(model, CONTEXT, 1), export_paged(model, SLOTS, PAGES, ROWS, SPAN))):
        chroma_amd.compile(graph, path).close()
    rules = random_rules(np.random.default_rng(7), 3001, 12)

    def expected(row, rule, k):
        adjusted = rule.apply(row)
        order = _select_host(as_float(adjusted), k, None)[1]
        return adjusted[order], order

    with Decoder(*map(Program, paths[:2])) as choosing, Decoder(*map(Program, paths[:2])) as full:
        for i, rule in enumerate(rules):
            k = (1, 7, 40)[i % 3]
            values, ids = choosing.append_top([i + 1], k, rules=rule)
            want_values, want_ids = expected(full.append([i + 1])[0], rule, k)
            np.testing.assert_array_equal(ids, want_ids)
            np.testing.assert_array_equal(values.view(np.uint8), want_values.view(np.uint8))
            if i % 4 == 0:  # the plain selection's captured graph between them
                values, ids = choosing.append_top([i + 2], 5)
                np.testing.assert_array_equal(ids, _select_host(as_float(full.append([i + 2])[0]), 5, None)[1])
    with PagedDecoder(Decoder(*map(Program, paths[:2])), Program(paths[2])) as choosing, \
            PagedDecoder(Decoder(*map(Program, paths[:2])), Program(paths[2])) as full:
        for decoder in (choosing, full):
            for prompt in ([1, 2, 3], [4], [5, 6, 7, 8]):
                decoder.add(prompt)
        for i in range(4):
            tokens = {2: i, 0: i + 10, 1: i + 20}
            chosen = {sequence: rules[3 * i + sequence] for sequence in ((0, 1, 2) if i % 2 else (1,))}
            values, ids = choosing.step_top(tokens, 6, rules=chosen)
            for row, sequence, got_values, got_ids in zip(full.step(tokens), tokens, values, ids):
                want_values, want_ids = expected(row, chosen.get(sequence, TokenRules()), 6)
                np.testing.assert_array_equal(got_ids, want_ids)
                np.testing.assert_array_equal(got_values.view(np.uint8), want_values.view(np.uint8))


def test_run_top_adjusted_refuses_no_rules():
    lib, error = native.library(), ctypes.create_string_buffer(256)
    status = lib.chroma_hip_run_top_adjusted(None, None, None, 0, 0, 1, 1, None, 1, None, None, error, len(error))
    assert status == native.RUNTIME_ERROR and b"null rules" in error.value
