"""Arguments of the operators around the pick and of the serving loop's requests, on the CPU. No GPU calls."""
import numpy as np
import pytest

from test_logits_capi import ADJUST, OTHER, X, refused

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


@pytest.mark.parametrize("bad", [V.Penalty(repeat=0.0), V.Penalty(repeat=-1.0), V.Penalty(repeat=float("inf")),
                                 V.Penalty(presence=float("nan")), V.Penalty(frequency=-float("inf"))])
def test_per_row_penalties_are_checked_as_shared_ones_are(bad):
    with pytest.raises(V.VsmpError, match="finite, repeat above 0"):
        V.to_device_penalties([V.Penalty(1.2, 0.5, 0.25, 8), bad], "cpu")
    with pytest.raises(V.VsmpError, match="finite, repeat above 0"):
        V.to_device_penalties(np.array([(bad.repeat, bad.presence, bad.frequency, 0)], V.PENALTY_DTYPE), "cpu")
    with pytest.raises(V.VsmpError, match="finite, repeat above 0"):
        decode.Request([1], decode.Opts(), penalty=bad)
    assert V.to_device_penalties([], "cpu").numel() == 0


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_adjust_refuses_per_row_penalties_off_their_alignment(shift):
    assert "per-row penalties" in refused("vsmp_adjust_logits", ADJUST, pen=OTHER + shift, per_row=1)
