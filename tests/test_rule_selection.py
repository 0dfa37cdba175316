"""Selection of tokens from adjusted logits over many steps (``run_top`` with rules): histories that grow, rules whose rows
lie apart, plain selections between them; and what the runtime refuses for the paged cache.

CPU: the runtime itself, built over a stand-in for HIP (``runtime_stub.cpp``) that counts what it allocates and captures.
GPU (marked): compiled programs against the host rule."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest
import torch

import chroma_amd
from chroma_amd import TokenRules
from chroma_amd._src import host, native
from chroma_amd._src.decoder import _select_host
from chroma_amd._src.program import NativeModel
from chroma_amd._src.rules import pack
from tests.conftest import ROOT
from tests.helpers import Function, as_float, numpy_of
from tests.test_paged_decoder import SLOTS, fake_paged_decoder, small_model

gpu = pytest.mark.gpu


class StubModel(NativeModel):
    """A program of one kernel that hands its input rows [rows, width] on as output 0."""

    def __init__(self, library, directory, rows, width):
        size = rows * width * 4
        room = -(-size // 256) * 256
        (directory / "weights.bin").write_bytes(b"")
        (directory / "model.plan").write_text("\n".join([
            "chroma-hip-plan 2", "signature none", "code_object none", "weights_file weights.bin", f"arena {2 * room + 1024}", "weights 0",
            f"error {2 * room}", f"input 0 0 {size}", f"output 0 {room} {size}", f"launch copy_{size} 1 1 1 64 0 2 0 {room}", ""]))
        spec = [{"name": "logits", "shape": [rows, width], "dtype": "float32"}]
        self.counted = library
        super().__init__(directory, spec, spec)
        self.started = self.counts()[3]

    def counts(self):
        """[device allocations, page-locked allocations, instantiated graphs, plan kernels and moves run] so far."""
        values = np.zeros(4, np.int64)
        self.counted.stub_counts(values.ctypes.data_as(ctypes.c_void_p))
        return values


@pytest.fixture(scope="module")
def stub_library(tmp_path_factory):
    path = tmp_path_factory.mktemp("stub") / "libstub.so"
    sources = [native.RUNTIME_SOURCE, ROOT / "tests" / "runtime_stub.cpp"]
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-w", "-D__HIP_PLATFORM_AMD__",
                    f"-I{native.ROCM / 'include'}", *map(str, sources), "-o", str(path)], check=True)
    library = ctypes.CDLL(str(path))
    for name in ("chroma_hip_create", "chroma_hip_run", "chroma_hip_device_name", "chroma_hip_signature", "chroma_hip_destroy", "chroma_hip_run_top",
                 "chroma_hip_run_top_adjusted", "chroma_hip_cache_move_queued"):
        function, known = getattr(library, name), getattr(native.library(), name)
        function.argtypes, function.restype = known.argtypes, known.restype
    return library


@pytest.fixture
def stub_model(stub_library, tmp_path, monkeypatch):
    def make(rows, width):
        with monkeypatch.context() as patch:
            patch.setattr(native, "library", lambda: stub_library)
            return StubModel(stub_library, tmp_path, rows, width)

    monkeypatch.setattr(host, "empty", lambda shape, dtype: np.empty(shape, dtype))
    return make


def chosen(rows, rules, k):
    """The host rule: the ``k`` largest adjusted values of each row and their ids."""
    picked = [_select_host(rule.apply(row), k, None) for row, rule in zip(rows, rules)]
    return np.stack([values for values, _ in picked]), np.stack([ids for _, ids in picked])


def test_growing_histories_keep_their_buffers_and_the_captured_selection(stub_model):
    """200 steps whose histories grow by 300 ids each (10 KB to 2 MB): buffers move a logarithmic number of times, and the
    plain selections between them replay the graph that the first one captured."""
    model, rng = stub_model(4, 100), np.random.default_rng(1)
    texts = [list(rng.integers(0, 100, 17 * i)) for i in range(4)]
    first = None
    for step in range(200):
        logits = rng.normal(size=(4, 100)).astype(np.float32) * 4
        for text in texts:
            text.extend(rng.integers(0, 100, 300))
        rules = [TokenRules(text, 1.0 + 0.1 * i, 0.01 * i, 0.001 * i) for i, text in enumerate(texts)]
        values, ids = model.run_top([logits], [None], 0, 3, rules)
        want_values, want_ids = chosen(logits, rules, 3)
        np.testing.assert_array_equal(ids, want_ids)
        np.testing.assert_array_equal(values, want_values)
        if step % 10 == 0:
            values, ids = model.run_top([logits], [None], 0, 3)
            np.testing.assert_array_equal(ids, chosen(logits, [TokenRules()] * 4, 3)[1])
        if first is None:
            first = model.counts()
    grown = model.counts() - first
    # half as much again each time: log(2 MB / 64 KiB) / log(1.5) = 8.5 moves, one buffer of each kind
    assert grown[0] <= 9 and grown[1] <= 9 and grown[2] == 0, grown


def test_rules_whose_rows_lie_apart(stub_model):
    """Rows of the rules' arrays further apart than they are long; what lies between them is nobody's."""
    rows, width, k, rng = 3, 70, 4, np.random.default_rng(5)
    model = stub_model(rows, width)
    rules = [TokenRules(rng.integers(0, width, 5 + i), 1.5, 0.25, 0.125, rng.normal(size=width).astype(np.float32), rng.random(width) < 0.6) for i in range(rows)]
    arrays = pack(rules, width)
    spread = {name: np.full((rows, arrays[name].shape[1] + gap), fill, arrays[name].dtype)
              for name, gap, fill in (("history", 3, 9), ("bias", 13, np.nan), ("mask", 2, 0))}
    for name, room in spread.items():
        room[:, : arrays[name].shape[1]] = arrays[name]
    call = native.Adjust(**{name: spread.get(name, array).ctypes.data for name, array in arrays.items()})
    call.history_width = arrays["history"].shape[1]
    call.history_stride, call.bias_stride, call.mask_stride = (spread[name].shape[1] for name in ("history", "bias", "mask"))
    logits = rng.normal(size=(rows, width)).astype(np.float32)
    values, ids, error = np.zeros((rows, k), np.float32), np.zeros((rows, k), np.int64), ctypes.create_string_buffer(256)
    native.check(model._lib.chroma_hip_run_top_adjusted(
        model._handle, native.pointer_array([logits.ctypes.data]), native.pointer_array([None]), 0, native.FLOAT32, rows, width, ctypes.byref(call), k,
        values.ctypes.data, ids.ctypes.data, error, len(error)), error)
    want_values, want_ids = chosen(logits, rules, k)
    np.testing.assert_array_equal(ids, want_ids)
    np.testing.assert_array_equal(values, want_values)


def adjusted_status(model, rules, rows, width, **strides):
    """(status, message) of a direct call with packed ``rules``, some strides or extents replaced."""
    arrays = pack(rules, width)
    call = native.Adjust(**{name: None if array is None else array.ctypes.data for name, array in arrays.items()})
    call.history_stride = call.history_width = arrays["history"].shape[1]
    for name, value in strides.items():
        setattr(call, name, value)
    logits, values, ids = np.ones((rows, width), np.float32), np.zeros((rows, 1), np.float32), np.zeros((rows, 1), np.int64)
    error = ctypes.create_string_buffer(256)
    status = model._lib.chroma_hip_run_top_adjusted(model._handle, native.pointer_array([logits.ctypes.data]), native.pointer_array([None]), 0, native.FLOAT32,
                                                    rows, width, ctypes.byref(call), 1, values.ctypes.data, ids.ctypes.data, error, len(error))
    return status, error.value.decode()


@pytest.mark.parametrize("rows,changes,message", [
    (65536, {}, "65535 rows"), (2, dict(history_width=-1), "stride"), (2, dict(history_stride=1), "stride"), (2, dict(bias_stride=3), "stride"),
    (2, dict(bias_stride=-4), "stride"), (2, dict(history_width=2**61, history_stride=2**61), "out of range")])
def test_refused_rules_run_nothing(stub_model, rows, changes, message):
    model = stub_model(rows, 4)
    status, text = adjusted_status(model, [TokenRules([1, 2], 1.5, bias={3: 1.0})] * rows, rows, 4, **changes)
    assert status == native.RUNTIME_ERROR and message in text
    assert model.counts()[3] == model.started, "the plan ran"


@pytest.mark.parametrize("tokens", [{0: 1, 1: 2, 2: 3}, {2: 5}], ids=["a-free-slot", "idle-sequences"])
def test_slots_without_a_token_do_not_end_the_sharing_of_a_bias_and_a_mask(tokens, monkeypatch):
    """Rules that all sequences of a step share are laid out as one row, whatever the other slots of the step program hold."""
    decoder = fake_paged_decoder(small_model())
    for prompt in ([1, 2], [3], [4, 5, 6]):
        decoder.add(prompt)
    bias, allowed = np.linspace(-1, 1, 17).astype(np.float32), np.arange(17) % 3 == 0
    rules = {s: TokenRules([s, s + 1], 1.5, bias=bias, allowed=allowed) for s in tokens}
    run_top, seen = decoder._step.native.run_top, []

    def watched(inputs, outputs, index, k, given):
        seen.append(pack(given, 17))
        return run_top(inputs, outputs, index, k, given)

    monkeypatch.setattr(decoder._step.native, "run_top", watched)
    values, ids = decoder.step_top(tokens, 2, rules=rules)
    assert (ids % 3 == 0).all() and np.isfinite(values).all()
    assert len(seen[0]["history"]) == SLOTS and seen[0]["bias"].shape == (1, 17) and seen[0]["mask"].shape == (1, 1)
    # a sequence with a token and without rules keeps its plain row, and a slot without a token then has one too
    if len(tokens) == 3:
        decoder.step_top(tokens, 2, rules={0: rules[0]})
        assert seen[1]["bias"].shape == (SLOTS, 17) and not seen[1]["bias"][1:].any() and (seen[1]["mask"][1:] == 0xFFFFFFFF).all()


@pytest.mark.parametrize("away", [None, ("to", "keys"), ("to", "values"), ("source", "keys"), ("source", "values")])
def test_queued_moves_of_memory_on_another_device_are_refused(stub_model, away):
    model, moves = stub_model(1, 4), np.array([[0, 1, 1]], dtype=np.int64)
    caches = {name: native.CacheRows(keys=base, values=base + 4096, rows=4, layer_pitch=64) for name, base in (("to", 1 << 20), ("source", 1 << 24))}
    if away is None:
        caches["source"].keys = 256  # what HIP does not know is left to the caller
        model.cache_move(caches["to"], caches["source"], 1, 16, moves)
        assert model.counts()[3] == model.started + 1
        return
    setattr(caches[away[0]], away[1], 1 << 60)
    with pytest.raises(RuntimeError, match="another device"):
        model.cache_move(caches["to"], caches["source"], 1, 16, moves)
    assert model.counts()[3] == model.started


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_growing_histories_on_the_device(tmp_path, dtype):
    """60 steps whose histories grow by 200 ids each, past the first room for rules, plain selections and their graph
    between them: values and ids bit for bit by the host rule (the same float operations)."""
    graph = torch.export.export(Function(lambda x: x * 0.5), (torch.zeros(3, 3001, dtype=dtype),))
    g, rng = torch.Generator().manual_seed(3), np.random.default_rng(3)
    texts, mask = [[], [1], [2, 3]], rng.random(3001) < 0.5
    with chroma_amd.compile(graph, tmp_path) as program:
        for step in range(60):
            x = (torch.randn(3, 3001, generator=g) * 8).to(dtype)
            rows = numpy_of(x * 0.5)
            for text in texts:
                text.extend(rng.integers(0, 3001, 200))
            rules = [TokenRules(text, 1.0 + 0.2 * i, 0.1 * i, 0.01 * i, None, mask if step % 2 else None) for i, text in enumerate(texts)]
            for given in ((rules, None) if step % 4 == 0 else (rules,)):
                values, ids = program.run_top_resident([numpy_of(x)], [None], 0, 5, rules=given)
                adjusted = [rule.apply(row) for rule, row in zip(given or [TokenRules()] * 3, rows)]
                for got_values, got_ids, row in zip(values, ids, adjusted):
                    order = _select_host(as_float(row), 5, None)[1]
                    np.testing.assert_array_equal(got_ids, order)
                    np.testing.assert_array_equal(got_values.view(np.uint8), row[order].view(np.uint8))
