"""GPU tests of drafted trees and their rules where a call meets what lies beside its own: rows next to
rows of another scale, requests that are refused, prompts among the nodes, empty lists of masks.

Tolerances are those of test_gpu_logit_rules.py; everything else is equal."""
import numpy as np
import pytest
import torch

from test_gpu_logit_rules import Rows
from test_gpu_paged import no_device_error

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- rows side by side ----
def falling(V, dtype, grammar, seed):
    """Rows each 100 below the one before, the best of a row below all of its neighbour's."""
    rows = Rows([3, 1, 2], V, dtype, history=(1, 30), biases=3, grammar=grammar, trees=True, seed=seed)
    T = len(rows.logits)
    rows.logits.copy_(rows.logits.float() / 4 + torch.arange(T, 0, -1, device="cuda")[:, None] * 100)
    return rows


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("V", [31, 97, 8191])
@pytest.mark.parametrize("grammar", [None, "some", "own"])
def test_a_row_chooses_among_its_own_tokens(cuda, dtype, V, grammar):
    """At every place of the first token in its 16 bytes, what lies before it is larger than any token of the
    row: the last logit of the row before, and for the first row what the memory holds there."""
    for offset in range(8):
        rows = falling(V, dtype, grammar, seed=V + offset)
        T = len(rows.logits)
        wide = torch.full((T * (V + 9) + 16,), 30000.0, dtype=rows.logits.dtype, device="cuda")
        full = Rows([200], 20000, dtype, seed=1)  # leaves large numbers wherever a chunk may lie on the chip
        full.logits.fill_(30000.0)
        for stride in (V, V + 1, V + 9):
            view = wide.as_strided((T, V), (stride, 1), offset)
            view.copy_(rows.logits)
            full.run()
            rows.check(*rows.run(logits=view))
        rows.check(*rows.run(out=view, logits=view))
    no_device_error()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("offset", [1, 7])
def test_nothing_is_left_beside_larger_rows(cuda, dtype, offset):
    """Biases of -infinity on all tokens but one, and on all: that one, or none."""
    V, T = 40, 6
    rows = falling(V, dtype, None, seed=offset)
    rows.drafted = None
    B = len(rows.counts)
    left = [[3], [], [39]]
    lists = [[v for v in range(V) if v not in left[b]] for b in range(B)]
    rows.bias = (np.concatenate([[0], np.cumsum([len(x) for x in lists])]), np.concatenate(lists),
                 np.full(sum(map(len, lists)), -np.inf, np.float32))
    wide = torch.full((T, V + offset), 30000.0, dtype=rows.logits.dtype, device="cuda")
    view = wide[:, offset:]
    view.copy_(rows.logits)
    out, chosen = rows.run(logits=view)
    rows.check(out, chosen)
    assert chosen.tolist() == [3, 3, 3, -1, 39, 39]
    no_device_error()
