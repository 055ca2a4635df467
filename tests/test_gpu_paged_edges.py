"""GPU tests of the serving operators at the edges of what their callers may
pass: what rows do not see, bounds that are not met, views, tokens outside
every request.  References and tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from test_gpu_paged import Batch, U, attention_reference, f64, i32, no_device_error, rope_reference, E32

pytestmark = pytest.mark.gpu


BEFORE = [
    # prefix, lens, queries, nq, nkv, hd, dtype, tokens before the first request, tokens after the last
    (0, [1, 30], [1, 1], 4, 2, 64, "fp16", 1, 0),
    (50, [9, 3], [1, 2], 8, 4, 128, "bf16", 3, 1),            # streamed prefix
    (300, [20] * 40, [1] * 40, 16, 8, 256, "fp16", 90, 5),    # whole tensor tiles before the first request
    (100, [150, 90], [150, 2], 16, 8, 64, "fp16", 37, 0),     # prompts in tiles that begin before it
]


@pytest.mark.parametrize("case", range(len(BEFORE)))
def test_tokens_before_the_first_request(cuda, case):
    """A batch that is a part of a longer list of tokens: those before it give out 0 and lse
    -infinity like those behind it, whatever the workspace holds."""
    prefix, lens, counts, nq, nkv, hd, dtype, before, after = BEFORE[case]
    batch = Batch(prefix, lens, counts, nq, nkv, hd, dtype, 16, seed=60 + case, padding=before + after)
    batch.starts = batch.starts + before
    out, lse = batch.run()
    no_device_error()
    batch.check(out, lse)
    assert (out[:before] == 0).all() and (lse[:before] == -float("inf")).all()
