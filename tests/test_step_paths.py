"""Steps of any number of tokens, and sampling, where the framework reaches them: the graph operator of chunk attention,
``PagedDecoder`` over an ``export_paged_chunk`` program, ``Sampling`` in the decoders, and the device operators in one run.

CPU: the operator's plain form, its lowering, ``PagedDecoder`` over a stand-in for device memory. GPU (marked): compiled
operators and whole models against the same."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import chroma_amd
from chroma_amd import Decoder, PagedDecoder, Program, Sampling, TokenRules
from chroma_amd._src import native
from chroma_amd._src.codegen.hip import HIPCodegen
from chroma_amd._src.compiler import lower_program
from chroma_amd._src.dtypes import float32_to_bf16
from chroma_amd._src.sampling import check_uniform, draw, pack
from chroma_amd.models.cached import export_cached
from chroma_amd.models.paged import export_paged, export_paged_chunk
from chroma_amd.ops import paged_chunk_attention
from oracle import compile_cpu
from tests.helpers import Function, as_float, numpy_of
from tests.test_decoder import FakeDevice
from tests.test_paged_decoder import CONTEXT, PAGES, ROWS, SLOTS, SPAN, FakePagedProgram, Twin, fake_paged_decoder, live_pages, small_model
from tests.test_step_operators import (chunk_inputs, chunk_reference, on_gpu, plain_chunk_call, plan_call, plan_reference, plan_room, queue, queue_in,
                                       row_settings, sample_call, sample_reference, store_call)

gpu = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
ROOM = 7  # tokens of a step
NAMES = ("q", "k_pages", "v_pages", "k_new", "v_new", "table", "lengths", "starts", "sinks")


# ------------------------------------------------------------------------------------------------ the operator
def within(got, inputs, **options):
    want, bound, taken = chunk_reference(**inputs, **options)
    got = got.double()
    assert torch.isfinite(got[taken]).all() and ((got - want).abs() <= bound)[taken].all()
    assert not got[~taken].any()


@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("window,first", [(0, 0), (5, 0), (7, 3)])
def test_plain_form_of_the_operator(window, first, fresh, dtype):
    inputs = chunk_inputs([3, 0, 6, 1], [5, 7, 20, 33], kv=2, group=3, dim=16, page=8, dtype=dtype, fresh=fresh, sinks=window == 0, seed=window)
    inputs["table"][2, 1] = len(inputs["k_pages"])
    inputs["lengths"][1] = -4
    inputs["lengths"][0] = 2  # stored: its first token lies before the text
    within(paged_chunk_attention(*(inputs[name] for name in NAMES), 0.25, window, first), inputs, window=window, first=first, scale=0.25)


def test_operator_refusals():
    inputs = chunk_inputs([2, 3], [5, 9], kv=2, group=2, dim=8, page=4, dtype=torch.float32)
    good = [inputs[name] for name in NAMES]
    paged_chunk_attention(*good, 1.0)
    for index, value, kind in ((0, good[0][0], ValueError), (1, good[1][:, :, :1], ValueError), (3, None, ValueError), (3, good[3][:1], ValueError),
                               (5, good[5].int(), TypeError), (5, good[5][:1], ValueError), (6, good[6][:1], ValueError), (6, good[6][:0], ValueError),
                               (7, good[7][:2], ValueError), (7, good[7].int(), TypeError), (8, good[8][:3], ValueError), (2, good[2].bfloat16(), TypeError),
                               (4, good[4].bfloat16(), TypeError), (8, good[8].double(), TypeError)):
        changed = list(good)
        changed[index] = value
        with pytest.raises(kind):
            paged_chunk_attention(*changed, 1.0)
    for window, first in ((-1, 0), (0, -1)):
        with pytest.raises(ValueError):
            paged_chunk_attention(*good, 1.0, window, first)


def exported(inputs, *, window=0, first=0):
    """(exported module, its arguments): the pages as layer 1 of 2, q and the new rows as expressions."""
    arguments = [inputs[name] for name in NAMES]
    for i in (1, 2):
        arguments[i] = torch.stack((torch.zeros_like(arguments[i]), arguments[i]))
    holes = [x is None for x in arguments]
    scale = inputs["q"].shape[-1] ** -0.5

    def call(*given):
        rest = iter(given)
        q, k, v, *others = (None if hole else next(rest) for hole in holes)
        pages = k.shape[1:]
        return paged_chunk_attention(q * 1.0, k[1:2].reshape(pages), v[1:2].reshape(pages), *others, scale, window, first)

    present = [x for x in arguments if x is not None]
    return torch.export.export(Function(call), tuple(present)), present


@pytest.mark.parametrize("shape,window,kernels", [
    (([3, 1], [40, 3], 2, 4, 64, 16), 0, ["tiles"]), (([3, 1], [4000, 3], 2, 4, 64, 16), 0, ["tiles", "combine"]),
    (([300, 1], [40, 3], 8, 4, 64, 16), 0, ["wide"]), (([130], [4000], 8, 8, 64, 16), 0, ["wide", "combine"]), (([130], [4000], 8, 8, 64, 16), 100, ["wide"])])
def test_lowering_cuts_by_the_rows_and_the_span(shape, window, kernels):
    counts, lengths, kv, group, dim, page = shape
    graph, _ = exported(chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=torch.bfloat16), window=window)
    source = lower_program(graph, HIPCodegen()).files["model.hip"]
    assert [name for name in ("tiles", "wide", "combine") if f"attention_chunk_{name}<" in source] == kernels


def test_compiled_calls_are_cut_as_the_library_cuts_them():
    """The scratch that the library asks for follows from the cut."""
    rng, lib = np.random.default_rng(3), native.library()
    split = set()
    for _ in range(400):
        tokens, sequences, kv = int(np.exp(rng.uniform(0, 9))), int(np.exp(rng.uniform(0, 4))), int(rng.choice([1, 2, 8]))
        group, dim, item = int(rng.choice([1, 5, 8])), int(rng.choice([8, 64, 80, 128, 256])), int(rng.choice([2, 4]))
        longest, window, fresh = int(np.exp(rng.uniform(0, 11))), int(rng.choice([0, 0, 500])), bool(rng.integers(2))
        waves, tiles, splits = HIPCodegen.chunk_cut(tokens, sequences, kv, group, dim, item, longest, fresh, window, 4)
        call = plain_chunk_call(tokens=tokens, sequences=sequences, kv_heads=kv, group=group, dim=dim, longest=longest, page_rows=16, table_stride=longest,
                                window=window, first=4, page_stride=16 * kv * dim, row_stride=kv * dim, head_stride=dim, q_stride=kv * group * dim,
                                out_stride=kv * group * dim, new_stride=kv * dim, dtype=native.BFLOAT16 if item == 2 else native.FLOAT32,
                                **({} if fresh else {"k_new": None, "v_new": None}))
        padded = next(n for n in (16, 32, 64, 128, 256) if n * item >= 64 and dim <= n)
        want = tiles * kv * splits * (32 * waves if waves else 16) * (padded + 2) * 4 if splits > 1 else 0
        assert lib.chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call)) == want
        split.add((waves, splits > 1))
    assert {(0, False), (0, True), (4, False), (4, True)} <= split


@gpu
@BOTH
@pytest.mark.parametrize("shape,window", [
    (([1, 0, 3, 17], [0, 5, 2, 64], 2, 3, 16, 16), 0), (([3, 1], [2500, 3], 1, 8, 64, 16), 0), (([300, 35], [64, 100], 8, 4, 128, 64), 0),
    (([150], [2500], 4, 16, 64, 16), 0), (([130, 7], [300, 40], 8, 8, 80, 12), 60)])
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
def test_compiled_operator(tmp_path, shape, window, fresh, dtype):
    counts, lengths, kv, group, dim, page = shape
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    inputs = chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=fresh, sinks=fresh, seed=dim, behind=5)
    graph, arguments = exported(inputs, window=window, first=2)
    with chroma_amd.compile(graph, tmp_path / "op") as program:
        for _ in range(3):
            got = program(*map(numpy_of, arguments))
        within(torch.from_numpy(as_float(got)), inputs, window=window, first=2)


# ------------------------------------------------------------------------------------------------ PagedDecoder
class ChunkTwin(Twin):
    def step(self, decoder, tokens):
        logits = decoder.step(tokens)
        assert len(logits) == len(tokens)
        for (sequence, some), row in zip(tokens.items(), logits):
            self.texts[sequence] += list(np.atleast_1d(some))
            self.check(sequence, row)
            assert decoder.position(sequence) == len(self.texts[sequence]) and len(decoder.pages(sequence)) == -(-len(self.texts[sequence]) // ROWS)


def walk(decoder, twin):
    """Prompts in steps of their own and beside decoded tokens, second turns, forks before and inside a page, ends."""
    a, logits = decoder.add([3, 1, 4, 1, 5, 9, 2, 6])  # two steps
    twin.texts[a] = [3, 1, 4, 1, 5, 9, 2, 6]
    twin.check(a, logits[0])
    b = decoder.begin()
    twin.texts[b] = []
    assert decoder.position(b) == 0 and decoder.pages(b) == []
    twin.step(decoder, {a: 5, b: [9, 2, 6]})
    twin.step(decoder, {b: [7, 7], a: [1, 2, 3, 4]})
    c, d = decoder.fork(b), decoder.begin()  # b holds 5 rows: its second page is shared until one of them writes
    twin.texts[c], twin.texts[d] = list(twin.texts[b]), []
    twin.step(decoder, {c: [2, 3, 4, 5], d: 8, b: [1]})
    assert decoder.pages(b)[0] == decoder.pages(c)[0] and decoder.pages(b)[1] != decoder.pages(c)[1]
    with pytest.raises(RuntimeError, match="holds 4 sequences"):
        decoder.add([1])
    decoder.free(a)
    live = live_pages(decoder)
    assert decoder.free_pages == PAGES - len(live)
    decoder.compact()
    assert live_pages(decoder) == set(range(len(live)))
    twin.step(decoder, {d: [1, 2, 3], b: np.array([4, 5]), c: (6,)})
    return b, c, d


def fake_chunk_decoder(model, pages=PAGES, kind=FakePagedProgram):
    return PagedDecoder(None, kind(export_paged_chunk(model, ROOM, SLOTS, pages, ROWS, SPAN), FakeDevice(1 << 22)))


def test_chunked_decoder_matches_the_model_on_the_host():
    model = small_model()
    with fake_chunk_decoder(model) as decoder:
        assert decoder.step_tokens == ROOM and decoder.vocab_size == 17
        b, _, d = walk(decoder, ChunkTwin(model, 2e-5, 2e-6))
        while decoder.position(d) + 5 <= SPAN * ROWS:
            decoder.step({d: [1] * 5})
        with pytest.raises(ValueError, match="more are not what the step program has pages for"):
            decoder.step({d: [1] * (SPAN * ROWS - decoder.position(d) + 1)})


def test_chunked_decoder_refuses_and_keeps_its_state():
    model = small_model()
    decoder = fake_chunk_decoder(model, pages=5)
    twin = ChunkTwin(model, 2e-5, 2e-6)
    a, _ = decoder.add([1, 2, 3, 4, 5, 6, 7])
    twin.texts[a] = [1, 2, 3, 4, 5, 6, 7]
    state = (decoder.pages(a), decoder.position(a), decoder.free_pages, decoder.sequences)

    def unchanged():
        assert (decoder.pages(a), decoder.position(a), decoder.free_pages, decoder.sequences) == state

    for tokens, kind in (({}, ValueError), ({a + 1: 1}, KeyError), ({a: 1.5}, TypeError), ({a: []}, ValueError), ({a: [[1]]}, ValueError),
                         ({a: [1, 17]}, IndexError), ({a: -1}, IndexError), ({a: [0] * (ROOM + 1)}, ValueError)):
        with pytest.raises(kind):
            decoder.step(tokens)
        unchanged()
    for prompt, kind in (([], ValueError), ([1] * (SPAN * ROWS + 1), ValueError), ([1] * 9, RuntimeError), ([17], IndexError), ([0.5], TypeError),
                         ([1, 17], IndexError)):
        with pytest.raises(kind):
            decoder.add(prompt)
        unchanged()
    with pytest.raises(IndexError):  # in its second step: the first one's pages go back
        fake = fake_chunk_decoder(model)
        free = fake.free_pages
        try:
            fake.add([1] * ROOM + [99])
        finally:
            assert fake.free_pages == free and fake.sequences == []
    with pytest.raises(RuntimeError, match="needs 3 pages, 2 are free"):
        decoder.step({a: [1] * 3, decoder.begin(): [1] * 4})
    twin.step(decoder, {a: [1, 2]})
    decoder.close()
    for call in (decoder.begin, lambda: decoder.add([1]), lambda: decoder.step({a: 1})):
        with pytest.raises(RuntimeError, match="closed"):
            call()


def test_decoders_and_step_programs_are_told_apart():
    model = small_model()
    device = FakeDevice(1 << 22)
    chunk, step = (FakePagedProgram(graph, device) for graph in (export_paged_chunk(model, ROOM, SLOTS, PAGES, ROWS, SPAN), export_paged(model, SLOTS, PAGES, ROWS, SPAN)))
    prompts = [FakePagedProgram(export_cached(model, CONTEXT, steps), device) for steps in (CONTEXT, 1)]
    with pytest.raises(ValueError, match="eight inputs"):
        PagedDecoder(None, step)
    with pytest.raises(ValueError, match="six inputs"):
        PagedDecoder(Decoder(*prompts, sliding_window=4), chunk)
    for part, index, shape in (("inputs", 3, [2, PAGES - 1, ROWS, 2, 8]), ("inputs", 6, [SLOTS]), ("inputs", 0, [ROOM, 1]), ("outputs", 1, [2, SLOTS, 2, 8]),
                               ("outputs", 0, [SLOTS + 1, 17])):
        spec = getattr(chunk, part)[index]
        kept, spec["shape"] = spec["shape"], shape
        with pytest.raises(ValueError, match="not exported by export_paged_chunk"):
            PagedDecoder(None, chunk)
        spec["shape"] = kept
    for extents in ((0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 1, 1, 0)):
        with pytest.raises(ValueError):
            export_paged_chunk(model, *extents)
    with fake_paged_decoder(model) as decoder:
        with pytest.raises(RuntimeError, match="the decoder consumes the prompts"):
            decoder.begin()
        with pytest.raises(TypeError, match="must be integers"):
            decoder.step({decoder.add([1, 2])[0]: [1, 2]})


@gpu
@BOTH
def test_chunked_decoder_matches_the_model(tmp_path, dtype):
    model = small_model().to(dtype)
    tolerance = (2e-5, 2e-6) if dtype == torch.float32 else (0.03, 0.03)  # bfloat16: the framework's tolerance for small whole models
    with PagedDecoder(None, chroma_amd.compile(export_paged_chunk(model, ROOM, SLOTS, PAGES, ROWS, SPAN), tmp_path / "step")) as decoder:
        walk(decoder, ChunkTwin(model, *tolerance))


# ------------------------------------------------------------------------------------------------ sampling
def test_settings_are_checked():
    for changes in (dict(temperature=-0.1), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.1),
                    dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=2.0), dict(min_p=-1.0)):
        with pytest.raises(ValueError, match=next(iter(changes))):
            Sampling(**changes)
    for value in (-1e-9, 1.0, math.nan):
        with pytest.raises(ValueError, match="uniform"):
            check_uniform(value)
    assert check_uniform(1 - 2.0**-40) == np.float32(1 - 2.0**-24)
    arrays = pack([Sampling(), Sampling(0.5, 2**60, 0.9, 0.1)], [0.25, 0.5])
    assert arrays["top_k"].tolist() == [0, 2**31] and arrays["temperature"].dtype == np.float32


def sampling_of(settings, r):
    return Sampling(max(0.0, float(settings["temperature"][r])), min(max(0, int(settings["top_k"][r])), 2**30), float(settings["top_p"][r]),
                    float(settings["min_p"][r]))


@BOTH
@pytest.mark.parametrize("width", [1, 2, 63, 900, 5000])
def test_drawing_on_the_host(width, dtype):
    rows = 60
    x = (torch.randn(rows, width, generator=torch.Generator().manual_seed(width)) * 3).to(dtype)
    x[10:20] = torch.randint(-2, 3, (10, width), generator=torch.Generator().manual_seed(1)).to(dtype)
    settings = row_settings(rows, seed=width)
    for r, (token, logprob, nearest) in enumerate(sample_reference(x, **settings)):
        if not 0 < nearest < 1e-9:
            got, share = draw(numpy_of(x[r]), sampling_of(settings, r), float(settings["uniform"][r]))
            assert got == token
            assert share == pytest.approx(logprob, rel=1e-9, abs=1e-7)
    assert draw(np.full(5, -np.inf, np.float32), Sampling(), 0.5) == (-1, -math.inf)
    assert draw(np.array([1, np.nan, np.inf, np.nan], np.float32), Sampling(), 0.5)[0] == 1
    assert draw(np.array([1, np.inf, np.inf, 0], np.float32), Sampling(), 0.75) == (2, pytest.approx(math.log(0.5)))


def near_places():
    """(row, random number, token) where the drawn place is the last of its token, in sums past 2^53: of n equal logits and a small
    one, u n is 1 below a multiple of 2^24, and the small weight's share lifts the place to 1 below that token's end."""
    found = []
    for n in range(2001, 12001, 2):
        u = -pow(n, -1, 2**24) % 2**24
        x = np.float32(math.log((2**20 - 1) * 2**24 / u) - 44 * math.log(2))
        small = int(np.rint(math.exp(float(x)) * 2.0**44))
        place = u * (n * 2**44 + small) >> 24
        if place % 2**44 == 2**44 - 1 and place >= 2**54 and len(found) < 8:
            found.append((np.append(np.zeros(n, np.float32), x), u / 2**24, place >> 44))
    return found


def test_places_next_to_a_border_past_53_bits():
    cases = near_places()
    assert len(cases) == 8
    for row, u, token in cases:
        assert draw(row, Sampling(), u)[0] == token


@gpu
def test_places_next_to_a_border_past_53_bits_on_the_device():
    for row, u, token in near_places():
        x, uniform = torch.from_numpy(row).cuda()[None], torch.tensor([u], device="cuda")
        ids, logprobs = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
        queue_in("chroma_hip_rows_sample", sample_call(x, ids, logprobs, uniform=uniform))
        assert int(ids) == token


def test_sampling_of_a_decoder_on_the_host(tmp_path):
    model = small_model()
    programs = [compile_cpu(export_cached(model, CONTEXT, steps), tmp_path / f"p{steps}") for steps in (CONTEXT, 1)]
    twins = [compile_cpu(export_cached(model, CONTEXT, steps), tmp_path / f"t{steps}") for steps in (CONTEXT, 1)]
    rules = TokenRules(history=[1, 2], repetition=1.5, allowed=range(3, 12))
    with Decoder(*programs, sliding_window=4) as decoder, Decoder(*twins, sliding_window=4) as twin:
        for i, sampling in enumerate((Sampling(), Sampling(0.0), Sampling(0.7, 5, 0.9, 0.01))):
            want = draw(rules.apply(twin.append([i, 4])[0]), sampling, 0.3 * i)
            assert decoder.append_sample([i, 4], sampling, uniform=0.3 * i, rules=rules) == want
        with pytest.raises(TypeError, match="Sampling"):
            decoder.append_sample([1], {"temperature": 1.0}, uniform=0.1)
        with pytest.raises(ValueError, match="uniform"):
            decoder.append_sample([1], uniform=1.0)
        with pytest.raises(IndexError):
            decoder.append_sample([1], uniform=0.5, rules=TokenRules(history=[99]))
        assert decoder.position == twin.position


class SamplingNative(type(fake_paged_decoder(small_model())._step._model)):
    def run_sample(self, inputs, outputs, index, sampling, uniform, rules=None):
        self.run(inputs, outputs, resident=True)
        rows = self.device.view(self.outputs[index], self.oracle.outputs[index])
        chosen = [draw(row if rules is None else rules[i].apply(row), sampling[i], uniform[i]) for i, row in enumerate(rows)]
        return np.array([token for token, _ in chosen]), np.array([logprob for _, logprob in chosen], dtype=np.float32)


class SamplingProgram(FakePagedProgram):
    def __init__(self, graph, device) -> None:
        super().__init__(graph, device)
        self._model.__class__ = SamplingNative


def sampled_steps(decoder, twin, room):
    """``step_sample`` against ``draw`` on the logits of a twin's ``step``."""
    rng = np.random.default_rng(0)
    for one in (decoder, twin):
        for prompt in ([3, 1, 4], [5], [9, 2, 6, 5]):
            one.add(prompt)
    plain = [Sampling(), Sampling(0.0), Sampling(0.6, 6, 0.95, 0.02), Sampling(1.3, 0, 0.5)]
    for i in range(6):
        tokens = {s: (list(rng.integers(0, 17, 1 + i % 2)) if room else int(rng.integers(0, 17))) for s in ((2, 0), (0, 1, 2), (1,))[i % 3]}
        uniform = {s: float(rng.random()) for s in tokens}
        sampling = plain[i % 4] if i % 2 else {s: plain[(i + s) % 4] for s in list(tokens)[1:]}
        rules = {list(tokens)[0]: TokenRules(history=[1, 2, 3], presence=1.0, allowed=range(2, 16))} if i in (2, 3, 5) else None
        ids, logprobs = decoder.step_sample(tokens, uniform, sampling, rules=rules)
        for s, row, token, logprob in zip(tokens, twin.step(tokens), ids, logprobs):
            row = (rules or {}).get(s, TokenRules()).apply(row)
            one = sampling.get(s, Sampling()) if isinstance(sampling, dict) else sampling
            want = draw(row, one, uniform[s])
            assert int(token) == want[0] and float(logprob) == pytest.approx(want[1], rel=2e-7, abs=2e-7)


@pytest.mark.parametrize("room", [0, ROOM], ids=["token", "chunk"])
def test_sampled_steps_on_the_host(room, monkeypatch):
    model = small_model()
    if room:
        decoder, twin = fake_chunk_decoder(model, kind=SamplingProgram), fake_chunk_decoder(model)
    else:
        decoder, twin = fake_paged_decoder(model), fake_paged_decoder(model)
        decoder._step._model.__class__ = SamplingNative
    sampled_steps(decoder, twin, room)
    state = (decoder.position(0), decoder.free_pages)
    for arguments, kind in ((({0: 1}, {}), KeyError), (({0: 1}, {0: 0.5, 1: 0.5}), KeyError), (({0: 1}, {0: 1.0}), ValueError), (({0: 1}, {0: 0.5}, {1: Sampling()}), KeyError),
                            (({0: 1}, {0: 0.5}, 0.7), TypeError), (({9: 1}, {9: 0.5}), KeyError), (({0: 17}, {0: 0.5}), IndexError)):
        with pytest.raises(kind):
            decoder.step_sample(*arguments)
        assert (decoder.position(0), decoder.free_pages) == state
    with pytest.raises(KeyError):
        decoder.step_sample({0: 1}, {0: 0.5}, rules={1: TokenRules()})


@gpu
@BOTH
def test_sampling_on_the_device(tmp_path, dtype):
    """``append_sample`` and ``step_sample`` against the host rule on the logits that a twin downloads."""
    model = small_model().to(dtype)
    graphs = (export_cached(model, CONTEXT, CONTEXT), export_cached(model, CONTEXT, 1), export_paged(model, SLOTS, PAGES, ROWS, SPAN),
              export_paged_chunk(model, ROOM, SLOTS, PAGES, ROWS, SPAN))
    paths = [tmp_path / name for name in ("prefill", "one", "step", "chunk")]
    for path, graph in zip(paths, graphs):
        chroma_amd.compile(graph, path).close()
    rng = np.random.default_rng(4)
    with Decoder(*map(Program, paths[:2]), sliding_window=4) as decoder, Decoder(*map(Program, paths[:2]), sliding_window=4) as twin:
        for i in range(8):
            tokens, u = list(rng.integers(0, 17, 1 + i % 3)), float(rng.random())
            sampling = (Sampling(), Sampling(0.0), Sampling(0.8, 4, 0.9, 0.05))[i % 3]
            rules = None if i % 2 else TokenRules(history=tokens, repetition=1.3, bias={int(tokens[0]): -2.0})
            row = twin.append(tokens)[0]
            token, logprob = decoder.append_sample(tokens, sampling, uniform=u, rules=rules)
            want = draw(row if rules is None else rules.apply(row), sampling, u)
            assert token == want[0] and logprob == pytest.approx(want[1], rel=2e-7, abs=2e-7)
            if i == 4:  # a selection between them
                np.testing.assert_array_equal(decoder.append_top([3], 2)[1], twin.append_top([3], 2)[1])
    for room, pair in ((0, paths[2]), (ROOM, paths[3])):
        decoders = [PagedDecoder(None if room else Decoder(*map(Program, paths[:2]), sliding_window=4), Program(pair)) for _ in range(2)]
        sampled_steps(*decoders, room)
        for decoder in decoders:
            decoder.close()


@gpu
def test_sampling_of_a_program_refuses(tmp_path):
    program = chroma_amd.compile(torch.export.export(Function(lambda x: (x * 2.0, x.sum(-1))), (torch.zeros(3, 50),)), tmp_path / "rows")
    x = np.random.default_rng(0).normal(size=(3, 50)).astype(np.float32)
    settings = [Sampling(), Sampling(0.0), Sampling(0.5, 3)]
    ids, logprobs = program.run_sample_resident([x], [None, None], 0, settings, [0.1, 0.2, 0.9])
    for r in range(3):
        want = draw(x[r] * 2, settings[r], [0.1, 0.2, 0.9][r])
        assert ids[r] == want[0] and logprobs[r] == pytest.approx(want[1], rel=2e-7, abs=2e-7)
    for arguments, kind, message in ((([x], [None, None], 0, settings[:2], [0.1, 0.2, 0.9]), ValueError, "for 3 rows"),
                                     (([x], [None, None], 0, settings, [0.1, 0.2]), ValueError, "for 3 rows"),
                                     (([x], [None, None], 0, settings, [0.1, 0.2, 1.0]), ValueError, "uniform"),
                                     (([x], [None, None], 0, settings, [0.1, 0.2, 0.3], [TokenRules()]), ValueError, "1 rules for 3 rows")):
        with pytest.raises(kind, match=message):
            program.run_sample_resident(*arguments)
    lib, error, model = native.library(), ctypes.create_string_buffer(256), program.native
    call, token, logprob = native.Sample(), np.zeros(3, np.int64), np.zeros(3, np.float32)
    uniform = np.full(3, 0.5, np.float32)
    call.uniform = uniform.ctypes.data
    ins, outs = model._pointers([x], [None, None], True)

    def run(index=0, dtype=native.FLOAT32, rows=3, width=50, settings=call, rules=None):
        return lib.chroma_hip_run_sample(model._handle, ins, outs, index, dtype, rows, width, rules, None if settings is None else ctypes.byref(settings),
                                         token.ctypes.data, logprob.ctypes.data, error, len(error))

    assert run() == native.OK
    for changes, message in ((dict(index=2), b"output index"), (dict(index=-1), b"output index"), (dict(dtype=7), b"dtype"), (dict(rows=2), b"byte size"),
                             (dict(rows=0), b"65535 rows"), (dict(width=0), b"524288"), (dict(rows=2**40), b"65535 rows"), (dict(settings=None), b"null settings"),
                             (dict(settings=native.Sample()), b"null uniform"), (dict(rules=ctypes.byref(native.Adjust(history=4096, history_width=-1))), b"stride")):
        assert run(**changes) == native.RUNTIME_ERROR and message in error.value, changes
    assert run() == native.OK
    program.close()


# ------------------------------------------------------------------------------------------------ the operators in one run
@gpu
@BOTH
def test_a_serving_loop_on_the_device(dtype):
    """Plan, store, attend, sample as one captured step, replayed: the host reads nothing between the replays. A stand-in for a
    model: queries, keys and values are rows of tables by token and position, logits the first head's result times a matrix."""
    g = torch.Generator().manual_seed(8)
    n, kv, group, dim, page, span, pages, room, vocabulary, steps = 5, 2, 4, 32, 8, 12, 50, 24, 9000, 6

    def values(*shape):
        return torch.randn(*shape, generator=g).to(dtype)

    width = kv * (group + 2) * dim
    fused, head = values(vocabulary, width), values(dim, vocabulary)
    counts, free = torch.tensor([6, 1, 0, 9, 4]), torch.randperm(pages, generator=g)
    uniform, prompts = torch.rand(steps, n, generator=g), torch.randint(0, vocabulary, (steps, room), generator=g)
    settings = row_settings(n, seed=3)
    settings.pop("uniform")
    device = on_gpu({"fused": fused, "head": head, "counts": counts, "free": free, "uniform": uniform[0].clone(), "ids": prompts[0].clone(),
                     "table": torch.full((n, span), -1), "lengths": torch.zeros(n, dtype=torch.int64), "cursor": torch.zeros(1, dtype=torch.int64),
                     "keys": torch.zeros(pages, page, kv, dim, dtype=dtype), "values": torch.zeros(pages, page, kv, dim, dtype=dtype),
                     "tokens": torch.zeros(n, dtype=torch.int64), "logprobs": torch.zeros(n), **settings})
    made, out = plan_room(n, room), torch.zeros(room, kv, group, dim, dtype=dtype, device="cuda")
    rows = torch.zeros(room, width, dtype=dtype, device="cuda")
    logits = torch.zeros(n, vocabulary, dtype=dtype, device="cuda")
    size = dim * kv * (4 if dtype == torch.float32 else 2)
    kept = {}

    def step():
        stream = torch.cuda.current_stream().cuda_stream
        queue("chroma_hip_paged_plan", plan_call({**device}, made, tokens=room, pages=pages, page=page), stream)
        torch.index_select(device["fused"], 0, device["ids"], out=rows)
        q, k, v = rows.split([kv * group * dim, kv * dim, kv * dim], 1)
        cache = [device[name].view(torch.uint8).view(1, pages * page, size) for name in ("keys", "values")]
        new = [x.view(torch.uint8).unsqueeze(0) for x in (k, v)]
        queue("chroma_hip_cache_store", store_call(*cache, *new, made["slots"]), stream)
        call = native.PagedChunk(
            q=q.data_ptr(), k_pages=device["keys"].data_ptr(), v_pages=device["values"].data_ptr(), table=device["table"].data_ptr(),
            lengths=made["new_lengths"].data_ptr(), starts=made["starts"].data_ptr(), out=out.data_ptr(), tokens=room, sequences=n, kv_heads=kv, group=group,
            dim=dim, pages=pages, page_rows=page, page_stride=page * kv * dim, row_stride=kv * dim, head_stride=dim, q_stride=width, out_stride=kv * group * dim,
            table_stride=span, longest=span * page, scale=dim**-0.5, dtype=native.FLOAT32 if dtype == torch.float32 else native.BFLOAT16)
        kept["attention"] = queue_in("chroma_hip_paged_chunk_attention", call, stream, kept.get("attention"))
        last = out[:, 0, 0].index_select(0, (made["starts"][1:] - 1).clamp(min=0))
        torch.mm(last, device["head"], out=logits)
        sample = sample_call(logits, device["tokens"], device["logprobs"], uniform=device["uniform"], **{name: device[name] for name in settings})
        kept["sample"] = queue_in("chroma_hip_rows_sample", sample, stream, kept.get("sample"))
        device["lengths"].copy_(made["new_lengths"])
        device["cursor"].copy_(made["taken"])

    step()  # (the library's own buffers and workspaces)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for name in ("lengths", "cursor", "keys", "values"):
        device[name].zero_()
    device["table"].fill_(-1)
    results = []
    for i in range(steps):
        device["uniform"].copy_(uniform[i])
        device["ids"].copy_(prompts[i])
        graph.replay()
        torch.cuda.synchronize()
        results.append({**{name: value.cpu().clone() for name, value in made.items()}, "out": out.cpu().clone(), "logits": logits.cpu().clone(),
                        "tokens": device["tokens"].cpu().clone(), "table": device["table"].cpu().clone()})
    lengths, cursor, table = [0] * n, 0, torch.full((n, span), -1)
    keys, cached = torch.zeros(pages, page, kv, dim, dtype=dtype), torch.zeros(pages, page, kv, dim, dtype=dtype)
    for i, got in enumerate(results):
        want = plan_reference(lengths, counts.tolist(), table, free, cursor, tokens=room, pages=pages, page=page)
        assert {name: got[name].tolist() for name in want} == want
        q, k, v = fused[prompts[i]].split([kv * group * dim, kv * dim, kv * dim], 1)
        for t, slot in enumerate(want["slots"]):
            if slot >= 0:
                keys[slot // page, slot % page], cached[slot // page, slot % page] = k[t].view(kv, dim), v[t].view(kv, dim)
        lengths, cursor, table = want["new_lengths"], want["taken"][0], torch.tensor(want["table"])
        exact, bound, taken = chunk_reference(q.reshape(room, kv, group, dim), keys, cached, table, torch.tensor(lengths), torch.tensor(want["starts"]))
        assert ((got["out"].double() - exact).abs() <= bound)[taken].all(), i
        for r, (token, _, nearest) in enumerate(sample_reference(got["logits"], uniform=uniform[i], **settings)):
            assert 0 < nearest < 1e-9 or int(got["tokens"][r]) == token, (i, r)
