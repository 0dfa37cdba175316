"""What the operators of a step of any number of tokens keep at the edges of their rules: rounding, extents past 64 bits, kernels
that only large calls take, and the host's part of a step."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from chroma_amd._src import native
from chroma_amd._src.codegen.hip import HIPCodegen
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


# ------------------------------------------------------------------------------------------------ kernels of large calls
def cut(inputs, window=0, first=0):
    """(waves of a tile, tiles, parts) of a call, by the rule that programs are compiled by."""
    tokens, kv, group, dim = inputs["q"].shape
    return HIPCodegen.chunk_cut(tokens, len(inputs["lengths"]), kv, group, dim, inputs["q"].element_size(), inputs["table"].shape[1] * inputs["k_pages"].shape[1],
                                inputs["k_new"] is not None, window, first)


def check_heads(inputs, heads, **options):
    """The whole call, its results of some KV heads against 64 bits."""
    group = inputs["q"].shape[2]
    some = {**inputs, "q": inputs["q"][:, heads], "k_pages": inputs["k_pages"][:, :, heads], "v_pages": inputs["v_pages"][:, :, heads]}
    for name in ("k_new", "v_new"):
        some[name] = None if inputs[name] is None else inputs[name][:, heads]
    some["sinks"] = None if inputs["sinks"] is None else inputs["sinks"].view(-1, group)[heads].reshape(-1)
    want, bound, taken = chunk_reference(**some, **options)
    device = on_gpu(inputs)
    out = torch.full(device["q"].shape, 7.0, dtype=device["q"].dtype, device="cuda")
    queue_in("chroma_hip_paged_chunk_attention", chunk_call(**device, out=out, **options))
    assert (out[~taken.cuda()] == 7.0).all() and torch.isfinite(out[taken.cuda()]).any()
    got, fine = out.cpu().double()[:, heads], torch.isfinite(want)
    assert torch.equal(got.isnan()[taken], want.isnan()[taken])
    assert torch.equal(got[taken][~fine[taken]].nan_to_num(0.5), want[taken][~fine[taken]].nan_to_num(0.5))
    assert (((got - want).abs() <= bound) | ~fine)[taken].all()
    return out


EIGHT_WAVES = [  # (tokens, cached rows, kv, group, dim, page)
    ([300, 0, 1, 70, 90, 3, 64], [40, 9, 130, 0, 65, 200, 64], 64, 1, 128, 16),
    ([300, 0, 1, 70, 90, 3, 64], [40, 9, 130, 0, 65, 200, 64], 64, 1, 104, 1),
    ([257, 0, 63], [33, 5, 129], 48, 8, 80, 12),
    ([40, 30, 200], [129, 64, 0], 26, 17, 72, 7),
    ([600], [90], 16, 16, 128, 64),
    ([130, 126, 2], [700, 0, 300], 64, 5, 120, 33),
]


@gpu
@pytest.mark.parametrize("window,first", [(0, 0), (100, 3), (70, 130), (1, 0)])
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("shape", EIGHT_WAVES, ids=lambda s: f"{sum(s[0])}after{max(s[1])}-{s[2]}x{s[3]}x{s[4]}-{s[5]}")
def test_tiles_of_eight_waves(shape, fresh, window, first):
    """Tiles of 256 rows (heads of 72 to 128, 512 of them or more): full, begun and of empty sequences, whole rows of an operand and
    shorter ones, pages that end inside a block and pages of one row."""
    counts, lengths, kv, group, dim, page = shape
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    inputs = chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=torch.bfloat16, fresh=fresh, sinks=fresh, seed=dim + page)
    assert cut(inputs, window, first)[0] == 8
    check_heads(inputs, [0, kv - 1], window=window, first=first)


@gpu
@pytest.mark.parametrize("where", ["new", "window", "first"])
@pytest.mark.parametrize("dim", [128, 96])
def test_tiles_of_eight_waves_and_values_that_are_not_finite(where, dim):
    """A value of infinity or NaN in a row that some tokens of a tile see and others do not; bad pages and lengths behind the table."""
    inputs = chunk_inputs([200, 150], [200, 61], kv=90, group=3, dim=dim, page=16, dtype=torch.bfloat16, seed=dim)
    options = {} if where == "new" else {"window": 60, "first": 0 if where == "window" else 9}
    if where == "new":
        inputs["v_new"][20, 0, 3], inputs["v_new"][141, 1, 7], inputs["v_new"][341, 0, dim - 1] = math.inf, math.nan, -math.inf
    else:
        page, row = inputs["table"][0, 160 // 16], 160 % 16
        inputs["v_pages"][page, row, 0, 5], inputs["v_pages"][page, row, 1, 33] = math.nan, -math.inf
    inputs["table"][0, 3], inputs["table"][1, 0] = -1, len(inputs["k_pages"])
    assert cut(inputs, **options)[0] == 8
    out = check_heads(inputs, [0, 1, 63], **options)
    assert not torch.isfinite(out[:350]).all()


LARGE_TILES = [  # what the tiles of 128 rows had no test of: one head of a KV head, pages of one row, both
    ([300, 40, 1], [64, 0, 129], 40, 1, 64, 16), ([150, 90], [65, 33], 9, 6, 40, 1), ([200, 0, 70], [1, 64, 63], 60, 1, 104, 1), ([140, 60], [90, 3], 44, 1, 256, 1)]


@gpu
@pytest.mark.parametrize("window,first", [(0, 0), (50, 3)])
@pytest.mark.parametrize("shape", LARGE_TILES, ids=lambda s: f"{sum(s[0])}after{max(s[1])}-{s[2]}x{s[3]}x{s[4]}-{s[5]}")
def test_large_tiles_of_one_head_and_pages_of_one_row(shape, window, first):
    counts, lengths, kv, group, dim, page = shape
    inputs = chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=torch.bfloat16, seed=dim + group)
    assert cut(inputs, window, first)[0] == 4
    check_heads(inputs, [0, kv // 2, kv - 1], window=window, first=first)


def test_tiles_of_eight_waves_are_never_split():
    """They are taken where there are 512 or more, as many as keys are split for; the library asks for no scratch."""
    rng, found = np.random.default_rng(5), 0
    for _ in range(3000):
        tokens, sequences, kv, group = int(np.exp(rng.uniform(3, 12))), int(np.exp(rng.uniform(0, 6))), int(rng.integers(1, 65)), int(rng.integers(1, 41))
        dim, longest, window = 8 * int(rng.integers(9, 17)), int(np.exp(rng.uniform(0, 14))), int(rng.choice([0, 300]))
        waves, _, parts = HIPCodegen.chunk_cut(tokens, sequences, kv, group, dim, 2, longest, True, window, 4)
        if waves != 8 or tokens * kv * group >= 2**26:
            continue
        found += 1
        call = plain_chunk_call(tokens=tokens, sequences=sequences, kv_heads=kv, group=group, dim=dim, longest=longest, page_rows=16, table_stride=longest,
                                window=window, first=4, page_stride=16 * kv * dim, row_stride=kv * dim, head_stride=dim, q_stride=kv * group * dim,
                                out_stride=kv * group * dim, new_stride=kv * dim)
        assert parts == 1 and native.library().chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call)) == 0
    assert found > 300
