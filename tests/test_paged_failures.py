"""``PagedDecoder`` when something goes wrong in the middle of a call, or when two threads use it: what it holds afterwards
are the sequences before the call, and the next calls answer as if it had not been made. (Stand-in for device memory.)"""

from __future__ import annotations

import threading

import pytest

from tests.test_paged_decoder import Twin, fake_paged_decoder, small_model


def broken(native, after):
    """``native.cache_move`` that fails after ``after`` calls; returns a function that mends it."""
    whole, calls = native.cache_move, iter(range(10**6))

    def move(*arguments):
        if next(calls) >= after:
            raise RuntimeError("cache_move: device lost")
        whole(*arguments)

    native.cache_move = move

    def mend():
        native.cache_move = whole

    return mend


def held(decoder):
    return {s: (decoder.pages(s), decoder.position(s)) for s in decoder.sequences}, decoder.free_pages


@pytest.mark.parametrize("after", [0, 1], ids=["copies", "new-rows"])
def test_a_step_whose_rows_cannot_be_stored_changes_nothing(after):
    """One sequence begins a page, one copies a shared page: the step fails at the copies or after them."""
    model = small_model()
    decoder, twin = fake_paged_decoder(model), Twin(model, 2e-5, 2e-6)
    a, b = decoder.add([3, 1, 4])[0], decoder.add([9, 2, 6, 5])[0]
    c = decoder.fork(b)
    twin.texts = {a: [3, 1, 4], b: [9, 2, 6, 5], c: [9, 2, 6, 5]}
    before = held(decoder)
    mend = broken(decoder._step.native, after)
    with pytest.raises(RuntimeError, match="device lost"):
        decoder.step({a: 1, b: 2, c: 3})
    assert held(decoder) == before
    mend()
    twin.step(decoder, {c: 7, b: 2, a: 1})
    twin.step(decoder, {a: 5, b: 6, c: 1})


def test_a_prompt_whose_rows_cannot_be_stored_takes_no_pages():
    model = small_model()
    decoder, twin = fake_paged_decoder(model), Twin(model, 2e-5, 2e-6)
    a = decoder.add([3, 1, 4, 1])[0]
    twin.texts[a] = [3, 1, 4, 1]
    before = held(decoder)
    mend = broken(decoder._step.native, 0)
    with pytest.raises(RuntimeError, match="device lost"):
        decoder.add([1, 2, 3, 4, 5])
    assert held(decoder) == before
    mend()
    b, logits = decoder.add([1, 2, 3, 4, 5])
    twin.texts[b] = [1, 2, 3, 4, 5]
    twin.check(b, logits[0])
    twin.step(decoder, {b: 6, a: 2})


def test_another_thread_cannot_use_the_decoder_in_the_middle_of_a_prompt():
    """A prompt's rows are taken from the decoder's cache after it consumed them: another user of the same decoder waits."""
    model = small_model()
    decoder, twin = fake_paged_decoder(model), Twin(model, 2e-5, 2e-6)
    prompts, append = decoder._decoder, decoder._decoder.append
    threads = []

    def consume(tokens):
        logits = append(tokens)

        def other():
            prompts.reset()
            append([16, 16, 16, 16, 16])

        threads.append(threading.Thread(target=other))
        threads[-1].start()
        threads[-1].join(0.5)  # ends here only if it is let in
        return logits

    prompts.append = consume
    a, logits = decoder.add([1, 2, 3, 4, 5])
    threads[0].join(30)
    assert not threads[0].is_alive() and prompts.position == 5
    prompts.append = append
    twin.texts[a] = [1, 2, 3, 4, 5]
    twin.check(a, logits[0])
    twin.step(decoder, {a: 6})
