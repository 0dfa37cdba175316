"""What the operators of a step of any number of tokens keep at the edges of their rules: rounding, extents past 64 bits, kernels
that only large calls take, and the host's part of a step."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from chroma_amd._src import native
from tests.test_paged_decoder import fake_paged_decoder, small_model
from tests.test_step_operators import HALF, chunk_call, chunk_inputs, chunk_reference, on_gpu, plain_chunk_call, queue_in, refused
from tests.test_step_paths import fake_chunk_decoder

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ weights
def widened(inputs):
    """The same values in float."""
    return {name: value.float() if isinstance(value, torch.Tensor) and value.is_floating_point() else value for name, value in inputs.items()}


@gpu
@pytest.mark.parametrize("shape", [([1] * 9, [70, 3, 129, 64, 0, 33, 5, 200, 1], 2, 8, 64, 16), ([16], [900], 2, 8, 64, 16), ([1, 3], [2500, 40], 1, 8, 128, 32),
                                   ([5, 9, 0, 2], [40, 300, 7, 90], 3, 3, 80, 12), ([2, 7], [150, 31], 2, 4, 256, 16), ([4, 1], [60, 61], 1, 20, 24, 7)],
                         ids=lambda s: f"{sum(s[0])}after{max(s[1])}-{s[2]}x{s[3]}x{s[4]}")
def test_few_tokens_meet_the_values_with_two_halves_of_their_weights(shape):
    """As ``paged_attention`` has it: beside a float evaluation of the same values and the result's rounding, at most 2^-16 of each
    weight is left out (half a step of bfloat16, twice)."""
    counts, lengths, kv, group, dim, page = shape
    inputs = chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=torch.bfloat16, seed=sum(counts) + dim)
    same = widened(inputs)
    want, bound, taken = chunk_reference(**same)  # (its bound: of a float evaluation, half a step of float included)
    spread, _, _ = chunk_reference(**{**same, "v_pages": same["v_pages"].abs(), "v_new": same["v_new"].abs()})
    bound = bound + HALF[torch.bfloat16] * (want.abs() + bound) + 2.0**-16 * spread
    device = on_gpu(inputs)
    out = torch.zeros_like(device["q"])
    queue_in("chroma_hip_paged_chunk_attention", chunk_call(**device, out=out))
    assert ((out.cpu().double() - want).abs() <= bound)[taken].all()


# ------------------------------------------------------------------------------------------------ extents
@pytest.mark.parametrize("longest", [2**63 - 1, 2**63 - 5, 2**62, 2**31])
def test_lengths_near_the_end_of_64_bits_are_refused(longest):
    """Sums of the extents do not wrap on the way to the refusal (pages and a table row that would hold such a length)."""
    call = plain_chunk_call(longest=longest, page_rows=2**30, table_stride=2**34)
    with pytest.raises(RuntimeError, match="paged_chunk_attention: .*longest out of range"):
        refused("chroma_hip_paged_chunk_attention", call, 1 << 45, 1 << 30)
    assert native.library().chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call)) == 0


# ------------------------------------------------------------------------------------------------ the host's part of a step
def test_a_truth_value_is_a_token():
    """``True`` is an integer of Python's, and a step of single tokens takes it as such."""
    model = small_model()
    with fake_paged_decoder(model) as decoder:
        a, b = decoder.add([1, 2, 3])[0], decoder.add([1, 2, 3])[0]
        logits = decoder.step({a: True, b: 1})
        assert np.array_equal(logits[0], logits[1]) and decoder.position(a) == 4
        with pytest.raises(TypeError, match="must be integers"):
            decoder.step({a: 1.0})
    with fake_chunk_decoder(model) as decoder:
        a, b = decoder.add([1, 2, 3])[0], decoder.add([1, 2, 3])[0]
        logits = decoder.step({a: True, b: [1]})
        assert np.array_equal(logits[0], logits[1]) and decoder.position(a) == 4


@pytest.mark.parametrize("make", [fake_paged_decoder, fake_chunk_decoder], ids=["tokens", "chunks"])
def test_single_tokens_of_a_step_cost_no_arrays(make, monkeypatch):
    """A token of a sequence stays a number, and the page table's rows are written where a page joins them: arrays for every
    sequence doubled the host's part of a step (8 / 32 / 64 sequences of 2041 rows 64 / 204 / 380 us, and 106 / 340 / 642)."""
    model = small_model()
    with make(model) as decoder:
        a, b = decoder.add([1, 2, 3, 4])[0], decoder.add([5, 6, 7])[0]
        table = [list(row) for row in decoder._args[4]]
        calls, written = [], []
        kept, set_row = type(decoder)._tokens_of, decoder._set_row
        monkeypatch.setattr(type(decoder), "_tokens_of", staticmethod(lambda tokens: (calls.append(tokens), kept(tokens))[1]))
        monkeypatch.setattr(decoder, "_set_row", lambda sequence: (written.append(sequence), set_row(sequence)))
        decoder.step({a: 1, b: np.int64(2)})  # b begins a page (of 3 rows)
        decoder.step({b: 3, a: 4})
        decoder.step({a: 5})
        assert calls == [] and written == [b, a]
        after = [list(row) for row in decoder._args[4]]
        assert table != after and [row[: len(decoder.pages(s))] for row, s in zip(after, (a, b))] == [decoder.pages(a), decoder.pages(b)]
        assert all(page == -1 for row, s in zip(after, (a, b)) for page in row[len(decoder.pages(s)):])
