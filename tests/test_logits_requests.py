"""Arguments of the operators around the pick and of the serving loop's requests, on the CPU. No GPU calls."""
import pytest

from test_logits_capi import ADJUST, X, refused

import verbo_amd as V
from verbo_amd import decode


@pytest.mark.parametrize("prompt,prompt_len", [([], 1), ([1, 2], 3), ([1, 2], -1)])
def test_request_refuses_prompt_lengths_outside_the_prompt(prompt, prompt_len):
    with pytest.raises(V.VsmpError, match="prompt_len"):
        decode.Request(prompt, decode.Opts(), prompt_len=prompt_len)


@pytest.mark.parametrize("prompt,prompt_len", [([], 0), ([1, 2], 0), ([1, 2], 2)])
def test_request_takes_prompt_lengths_within_the_prompt(prompt, prompt_len):
    assert decode.Request(prompt, decode.Opts(), prompt_len=prompt_len).prompt_len == prompt_len


@pytest.mark.parametrize("change", [
    dict(ldi=250, ldo=250, out=X + 4 * 50),                # an output row begins inside a row of logits
    dict(ldi=180, ldo=180, out=X + 4 * 100),               # and ends inside the next one
    dict(ldi=250, ldo=251, out=X + 4 * 120),               # strides that drift apart
    dict(ldi=250, ldo=250, out=X - 4 * 500 + 4 * 50),      # from below
    dict(dtype=1, ldi=500, ldo=250, out=X + 2 * 98),       # 16-bit logits of the same stride in bytes
    dict(dtype=1, ldi=250, ldo=250, out=X + 4 * 120),
])
def test_adjust_refuses_outputs_that_overlap_rows_of_logits(change):
    assert "overlap" in refused("vsmp_adjust_logits", ADJUST, **change)
