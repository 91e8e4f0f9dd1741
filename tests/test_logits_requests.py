"""A serving loop's requests with penalties, and penalties on their way to the device, on the CPU. No GPU calls."""
import pytest

import verbo_amd as V
from verbo_amd import decode


@pytest.mark.parametrize("prompt,prompt_len", [([], 1), ([1, 2], 3), ([1, 2], -1)])
def test_request_refuses_prompt_lengths_outside_the_prompt(prompt, prompt_len):
    with pytest.raises(V.VsmpError, match="prompt_len"):
        decode.Request(prompt, decode.Opts(), prompt_len=prompt_len)


@pytest.mark.parametrize("prompt,prompt_len", [([], 0), ([1, 2], 0), ([1, 2], 2)])
def test_request_takes_prompt_lengths_within_the_prompt(prompt, prompt_len):
    assert decode.Request(prompt, decode.Opts(), prompt_len=prompt_len).prompt_len == prompt_len
