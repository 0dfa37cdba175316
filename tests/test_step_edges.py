"""What the operators of a step of any number of tokens keep at the edges of their rules: rounding, extents past 64 bits, kernels
that only large calls take, and the host's part of a step."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests.test_step_operators import HALF, chunk_call, chunk_inputs, chunk_reference, on_gpu, queue_in

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
