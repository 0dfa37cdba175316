"""The batched decoding operators where a rule on sizes chooses another kernel: logit adjustments over long spans, attention in
shares at every padded head dimension, two captured calls that both use scratch, the cut of compiled programs against the
C call's; and ``PagedDecoder`` over prompts of several calls, long texts in bfloat16 and two threads."""

from __future__ import annotations

import ctypes
import re
import threading

import numpy as np
import pytest
import torch

import chroma_amd
from chroma_amd import Decoder, PagedDecoder
from chroma_amd._src import native
from chroma_amd._src.codegen.hip import HIPCodegen
from chroma_amd._src.compiler import lower_program
from chroma_amd.models.cached import export_cached
from chroma_amd.models.paged import export_paged
from chroma_amd.ops import paged_attention
from tests.helpers import Function, random_transformer, small_config
from tests.test_batched_operators import adjust_inputs, attend, attention_call, check_adjust, check_attention, on_gpu, paged_inputs
from tests.test_decoder import FakeDevice
from tests.test_paged_decoder import (CONTEXT, PAGES, ROWS, SLOTS, SPAN, FakePagedProgram, Twin, fake_paged_decoder, small_model)

gpu = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


# ------------------------------------------------------------------------------------------------ logit adjustments
@gpu
@DTYPES
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in-place"])
@pytest.mark.parametrize("rows,width,history,bias,mask", [
    (800, 515, 40, "shared", "rows"), (768, 8192, 3, None, None), (110, 50001, 600, "rows", "rows"), (400, 8197, 5000, None, "shared"),
    (1000, 1, 2, "rows", "rows")])
def test_rows_adjust_over_long_spans(rows, width, history, bias, mask, in_place, dtype):
    """rows x ceil(width / 8192) of 768 and more take spans of 8192 ids."""
    assert rows * -(-width // 8192) >= 768
    x, inputs = adjust_inputs(rows, width, history, dtype, rows + width, bias=bias, mask=mask)
    check_adjust(x, inputs, in_place)


# ------------------------------------------------------------------------------------------------ attention
def workspace_bytes(call):
    return native.library().chroma_hip_paged_attention_workspace(ctypes.byref(call))


@gpu
@DTYPES
@pytest.mark.parametrize("window,first", [(0, 0), (2300, 70)])
@pytest.mark.parametrize("lengths,kv,group,dim,page", [
    ([4000, 1, 0], 2, 5, 128, 16), ([3100, 2600], 1, 16, 128, 64), ([5000, 30], 1, 20, 128, 7), ([3100, 0, 2600], 2, 3, 80, 16),
    ([2500, 2700], 1, 33, 80, 12), ([3000, 2000], 1, 2, 200, 16), ([3300], 4, 6, 48, 32), ([2600, 40], 1, 18, 24, 16)])
def test_paged_attention_in_shares(lengths, kv, group, dim, page, window, first, dtype):
    """Head dimensions that fill their padding and that do not, up to 16 query heads of a KV head and more, with the parts of
    a sequence in several shares."""
    inputs = paged_inputs(lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=bool(window), sinks=not window, seed=dim + group)
    assert workspace_bytes(attention_call(**inputs, out=torch.empty_like(inputs["q"]), window=window, first=first)) > 0
    check_attention(inputs, window=window, first=first)


@gpu
@DTYPES
def test_two_captured_calls_with_scratch_at_the_same_time(dtype):
    """Replays on two streams, each call with a workspace of its own, eager work between them."""
    inputs = [on_gpu(paged_inputs([4000, 3], kv=2, group=8, dim=64, page=16, dtype=dtype, seed=1)),
              on_gpu(paged_inputs([3200, 2800, 70], kv=1, group=8, dim=32, page=16, dtype=dtype, seed=2))]
    outs = [torch.empty_like(given["q"]) for given in inputs]
    calls = [attention_call(**given, out=out) for given, out in zip(inputs, outs)]
    graphs, kept, eager = [], [], []
    for call, out in zip(calls, outs):
        assert workspace_bytes(call) > 0
        attend(call)
        torch.cuda.synchronize()
        eager.append(out.clone())
    for call in calls:
        kept.append(torch.full((workspace_bytes(call),), 0xFF, dtype=torch.uint8, device="cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(call, torch.cuda.current_stream().cuda_stream, kept[-1])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, eager):
            assert torch.equal(out, want), turn
        attend(calls[turn % 2])
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], eager[turn % 2])


def test_compiled_programs_cut_as_the_c_call():
    """The same call through the compiler and through the C entry: whole sequences or shares, as many shares, as much scratch."""
    rng, seen = np.random.default_rng(11), set()
    for _ in range(40):
        kv, group, dim = [(1, 1, 8), (1, 8, 16), (2, 3, 24), (2, 20, 32), (8, 8, 64), (4, 7, 128), (1, 17, 80), (2, 2, 256)][rng.integers(8)]
        sequences, page, span = int(rng.integers(1, 70)), int(rng.choice([1, 7, 16, 64])), int(np.exp(rng.uniform(0, 6)))
        window, first = int(rng.choice([0, 0, 100, 2000])), int(rng.choice([0, 4, 3000]))
        dtype = [torch.float32, torch.bfloat16][rng.integers(2)]
        q, pages = torch.zeros(sequences, kv, group, dim, dtype=dtype), torch.zeros(3, page, kv, dim, dtype=dtype)
        table, lengths = torch.zeros(sequences, span, dtype=torch.int64), torch.zeros(sequences, dtype=torch.int64)

        def call(q, k, v, table, lengths):
            return paged_attention(q, k, v, None, None, table, lengths, None, 0.5, window, first)

        source = lower_program(torch.export.export(Function(call), (q, pages, pages.clone(), table, lengths)), HIPCodegen()).files["model.hip"]
        ranges = re.findall(r"attention_paged_shares<[^>]*, (\d+), \d+u, (?:true|false)>\(a, (\d+)u", source)
        assert len(re.findall("attention_paged_whole<", source)) == (not ranges)
        need = workspace_bytes(attention_call(q, pages, pages, table, lengths, torch.empty_like(q), window=window, first=first))
        got = 0 if not ranges else (int(ranges[0][1]) + sequences) * kv * group * (int(ranges[0][0]) + 2) * 4
        assert got == need, (sequences, kv, group, dim, page, span, window, first, dtype)
        seen.add(bool(ranges))
    assert seen == {True, False}


# ------------------------------------------------------------------------------------------------ PagedDecoder
PROMPTS = ([3, 1, 4, 1, 5, 9, 2, 6, 5], [2, 7, 1, 8], [1, 6, 1, 8, 0, 3, 3, 9], [5])  # of 9, 4, 8 and 1 tokens in calls of 4


def add_prompts(decoder, twin):
    for prompt in PROMPTS:
        sequence, logits = decoder.add(prompt)
        twin.texts[sequence] = list(prompt)
        twin.check(sequence, logits[0])
    twin.step(decoder, {s: s + 1 for s in decoder.sequences})
    twin.step(decoder, {s: s + 2 for s in decoder.sequences})


def test_prompts_of_several_calls():
    """Prompts longer than the prefill program's steps: their rows come from several calls, the last of one or more tokens."""
    model, device = small_model(), FakeDevice(1 << 22)
    programs = [FakePagedProgram(export_cached(model, CONTEXT, steps), device) for steps in (4, 1)]
    step = FakePagedProgram(export_paged(model, SLOTS, PAGES, ROWS, SPAN), device)
    add_prompts(PagedDecoder(Decoder(*programs, sliding_window=4), step), Twin(model, 2e-5, 2e-6))


@gpu
def test_prompts_of_several_calls_on_the_device(tmp_path):
    model = small_model()
    programs = [chroma_amd.compile(export_cached(model, CONTEXT, steps), tmp_path / f"p{steps}") for steps in (4, 1)]
    step = chroma_amd.compile(export_paged(model, SLOTS, PAGES, ROWS, SPAN), tmp_path / "step")
    with PagedDecoder(Decoder(*programs, sliding_window=4), step) as decoder:
        add_prompts(decoder, Twin(model, 2e-5, 2e-6))


@gpu
def test_long_texts_in_bfloat16(tmp_path):
    """Steps whose attention runs in shares, in bfloat16 (the framework's tolerance for small whole models)."""
    model = random_transformer(small_config(num_hidden_layers=2, head_dim=64, hidden_size=32, num_attention_heads=4, num_key_value_heads=2,
                                            sliding_window=50), seed=5, std=0.2).to(torch.bfloat16)
    context = 1700
    programs = [chroma_amd.compile(export_cached(model, context, steps), tmp_path / f"p{steps}") for steps in (context, 1)]
    step = chroma_amd.compile(export_paged(model, 3, 140, 16, 120), tmp_path / "step")
    assert "attention_paged_shares<" in (tmp_path / "step" / "model.hip").read_text()
    text, twin = (np.arange(context) * 7 % 17).tolist(), Twin(model, 0.03, 0.03)
    with PagedDecoder(Decoder(*programs, sliding_window=50), step) as decoder:
        a, logits = decoder.add(text)
        twin.texts[a] = list(text)
        twin.check(a, logits[0])
        b = decoder.fork(a)
        twin.texts[b] = list(text)
        twin.step(decoder, {a: 3, b: 4})
        twin.step(decoder, {b: 5, a: 1})


def test_two_threads_step_their_own_sequences():
    """Calls from two threads, each with sequences of its own that it extends, forks and ends: every answer is its text's."""
    model = small_model()
    decoder, failures = fake_paged_decoder(model), []

    def work(offset):
        try:
            twin = Twin(model, 2e-5, 2e-6)
            for turn in range(3):
                prompt = [(offset + turn + i) % 17 for i in range(2 + offset)]
                a, logits = decoder.add(prompt)
                twin.texts[a] = list(prompt)
                twin.check(a, logits[0])
                twin.step(decoder, {a: 1 + offset})
                b = decoder.fork(a)
                twin.texts[b] = list(twin.texts[a])
                for token in range(3):
                    twin.step(decoder, {b: token, a: token + offset})
                decoder.free(a)
                decoder.compact()
                twin.step(decoder, {b: 7})
                decoder.free(b)
        except BaseException as e:  # noqa: B902
            failures.append(e)

    threads = [threading.Thread(target=work, args=(offset,)) for offset in (0, 3)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(120)
    assert not failures and not any(thread.is_alive() for thread in threads)
    assert decoder.free_pages == PAGES and not decoder.sequences
