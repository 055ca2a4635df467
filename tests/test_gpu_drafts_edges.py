"""GPU tests of drafted trees and their rules where a call meets what lies beside its own: rows next to
rows of another scale, requests that are refused, prompts among the nodes, empty lists of masks.

Tolerances are those of test_gpu_logit_rules.py; everything else is equal."""
import numpy as np
import pytest
import torch

from test_gpu_draft_decoder import VOCAB, Round, make, model, padded  # noqa: F401 (model: a fixture)
from test_gpu_logit_rules import Rows
from test_gpu_paged import i32, no_device_error

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


# ---------------------------------------------------------- the whole step ----
def play_in_list_order(dec, cache, r, lens, refused=(), own_rows=False):
    """A round whose masks are given by token of the list, as its tokens and parents are."""
    live = [b for b in range(len(lens)) if len(r.tokens[b])]
    bits, rows = r.masks()
    if own_rows:  # a mask a token, most of them allowing everything
        bits = np.concatenate([bits, np.full_like(bits[:1], -1)])[rows + [-1] * (dec.T - len(rows))]
        rules = dict(allowed=torch.from_numpy(bits).cuda())
    else:
        rules = dict(allowed=torch.from_numpy(bits).cuda(), allowed_rows=padded(rows, dec.T))
    counts, new = dec.draft(i32(np.concatenate(r.tokens)), i32(np.concatenate(r.trees)),
                            i32([lens[b] + len(r.tokens[b]) if b in live else -1 for b in range(len(lens))]),
                            given=i32([len(k) for k in r.known]), rules=rules)
    torch.cuda.synchronize()
    counts, new, paths = counts.tolist(), new.cpu().numpy(), dec.paths.cpu().numpy()
    assert dec.draft_state.tolist()[2] == len(refused)
    for b in live:
        if b in refused:
            assert counts[b] == 0 and (new[b] == -1).all()
            continue
        path, fresh = r.expected(b)
        assert counts[b] == len(path) and paths[b, :len(path)].tolist() == path
        assert new[b, :len(fresh)].tolist() == fresh and (new[b, len(fresh):] == -1).all()
        lens[b] += len(path)
        r.known[b] = np.array(fresh[-1:])
    assert cache.seq_lens.tolist() == lens


@pytest.mark.parametrize("own_rows", [False, True])
@pytest.mark.parametrize("full", [[0], [1], [0, 2], [0, 1, 2, 3]])
def test_masks_stay_with_their_tokens_when_requests_are_refused(cuda, model, full, own_rows):  # noqa: F811
    """Requests whose tables have no room are refused, before and between others: these run under their own masks."""
    weights, _ = model
    rng = np.random.default_rng(sum(full) + 10 * len(full))
    dec, cache = make(weights, 4, 60, 4, 60, 4, 16)  # 16 positions a request
    lens = [0, 0, 0, 0]
    r = Round(rng, [rng.integers(VOCAB, size=14 if b in full else 3) for b in range(4)], (0, 0, 0, 0))
    play_in_list_order(dec, cache, r, lens, own_rows=own_rows)
    r = Round(rng, r.known, (5, 6, 4, 7))
    play_in_list_order(dec, cache, r, lens, refused=full, own_rows=own_rows)
    no_device_error()


def test_masks_for_too_few_tokens_are_refused(cuda, model):  # noqa: F811
    from edgeexpert_b200._lib import TFError
    weights, _ = model
    dec, cache = make(weights, 1, 8, 4, 8, 4, 4)
    ids, parents, targets = i32([1, 2, 3]), i32([-1, 0, 0]), i32([3])
    bits = i32(np.zeros((3, -(-VOCAB // 32))))
    for rules in (dict(allowed=bits[:2]), dict(allowed=bits, allowed_rows=i32([0, 1])), dict(allowed_rows=i32([0, 1, 2])),
                  dict(allowed=bits, allowed_rows=i32([[0, 1, 2]])), dict(allowed=bits, allowed_rows=i32([0, 1, 2]).cpu())):
        with pytest.raises(TFError):
            dec.draft(ids, parents, targets, rules=rules)
    assert cache.seq_lens.tolist() == [0]
    dec.draft(ids[:0], parents[:0], i32([-1]), rules=dict(allowed=bits))  # no tokens, nothing to do
    dec.draft(ids, parents, targets, rules=dict(allowed=bits))  # a row of the step is nobody's
    assert dec.tokens[:3].tolist() == [-1] * 3 and dec.counts.tolist() == [1]
    no_device_error()
