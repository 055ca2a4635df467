"""GPU tests of drafted trees and their rules where a call meets what lies beside its own: rows next to
rows of another scale, requests that are refused, prompts among the nodes, empty lists of masks.

Tolerances are those of test_gpu_logit_rules.py; everything else is equal."""
import numpy as np
import pytest
import torch

from test_gpu_draft_decoder import VOCAB, Round, make, model, padded  # noqa: F401 (model: a fixture)
from test_gpu_drafts import TreeBatch, flags, way, words_of
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


def test_masks_without_a_row(cuda):
    """No rows of allowed tokens are rows for nobody: refused, or, where rows are named, reported."""
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.sampling import LogitRules
    op, z = LogitRules(), torch.randn(3, 70, device="cuda")
    ws = torch.empty(op.workspace_bytes(3, 70, 3), dtype=torch.uint8, device="cuda")
    out, starts, nobody = torch.empty_like(z), i32([0, 1, 2, 3]), torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    with pytest.raises(TFError):
        op.encode(z, out, starts, ws, allowed=nobody)
    op.encode(z, out, starts, ws, allowed=nobody, allowed_rows=i32([-1, -1, -1]))
    torch.cuda.synchronize()
    assert torch.equal(out, z)
    no_device_error()
    op.encode(z, out, starts, ws, allowed=nobody, allowed_rows=i32([-1, 0, -1]))
    assert flags() and torch.equal(out, z)
    op.encode(z[:0], out[:0], i32([0, 0]), ws, allowed=nobody)
    no_device_error()


# ------------------------------------------------ prompts among the nodes ----
def prompts_as_history(rows, first):
    """The same rules with the first nodes' tokens in the history's prompt, and no tokens of their own."""
    n = np.minimum(first, rows.counts).clip(0)
    wide = np.full((len(n), rows.history.shape[1] + max(n)), -1)
    drafted = rows.drafted.copy()
    for b, k in enumerate(n):
        at, cut = rows.starts[b], rows.prompt[b]
        line = np.concatenate([rows.history[b, :cut], drafted[at:at + k], rows.history[b, cut:]])
        wide[b, :len(line)] = line
        drafted[at:at + k] = -1
    rows.history, rows.lens, rows.prompt, rows.drafted = wide, rows.lens + n, rows.prompt + n, drafted


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("counts,first,V", [([5, 9, 1, 1, 0, 7], [3, 1, 1, 0, 2, 99], 1000), ([60, 256], [40, -3], 97),
                                            ([12], [12], 20001)])
def test_first_nodes_that_are_a_prompt(cuda, dtype, counts, first, V):
    """The same bits as with those tokens in the history's prompt, and these are the definition's."""
    from edgeexpert_b200.sampling import LogitRules
    op, rows = LogitRules(), Rows(counts, V, dtype, history=(0, 20), prompt=0.3, biases=5, trees=True, seed=V)
    T, B = len(rows.logits), len(counts)
    f32 = [torch.from_numpy(x).cuda() for x in (rows.rep, rows.pres, rows.freq, rows.bias[2])]
    out, tokens = torch.full_like(rows.logits, 7.0), i32(np.full(T, 77))
    ws = torch.empty(rows.workspace(op, T), dtype=torch.uint8, device="cuda")
    op.encode(rows.logits, out, i32(rows.starts), ws, max_query=max(counts), history=i32(rows.history),
              history_lens=i32(rows.lens), prompt_lens=i32(rows.prompt), repetition=f32[0], presence=f32[1],
              frequency=f32[2], bias_starts=i32(rows.bias[0]), bias_tokens=i32(rows.bias[1]), bias_values=f32[3],
              token_ids=i32(rows.drafted), ancestors=words_of(rows.masks, -(-max(counts) // 32)), tokens=tokens,
              prompt_nodes=i32(first))
    prompts_as_history(rows, np.array(first))
    want, chosen = rows.run()
    rows.check(want, chosen)
    assert torch.equal(out, want) and torch.equal(tokens, chosen)
    no_device_error()


def test_prompt_nodes_refusals(cuda):
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.sampling import LogitRules
    op, z = LogitRules(), torch.zeros(2, 64, device="cuda")
    ws = torch.empty(op.workspace_bytes(2, 64, 2), dtype=torch.uint8, device="cuda")
    one = i32([1, 1])
    for bad in (dict(prompt_nodes=one), dict(prompt_nodes=one[:1], token_ids=one, ancestors=one[:, None]),
                dict(prompt_nodes=one.long(), token_ids=one, ancestors=one[:, None]),
                dict(prompt_nodes=one.cpu(), token_ids=one, ancestors=one[:, None])):
        with pytest.raises(TFError):
            op.encode(z, z, i32([0, 1, 2]), ws, **bad)
    no_device_error()


@pytest.mark.parametrize("given,prompt_nodes,asked", [([5, 1, 3], None, [5, 0, 3]), (None, None, [0, 0, 0]),
                                                      ([5, 1, 3], [5, 1, 0], [5, 1, 0])])
def test_a_prompt_in_a_step_is_no_output(cuda, model, given, prompt_nodes, asked):  # noqa: F811
    """Logits under penalties are the plain step's after fp32 steps of the definition: on a prompt's tokens the
    repetition penalty alone, on the others of a row's way all of them."""
    weights, _ = model
    rng = np.random.default_rng(3)
    counts = [9, 6, 7]
    trees = [np.concatenate([np.arange(g) - 1, rng.integers(g - 1, np.arange(g, n))])
             for g, n in zip(given or [1, 1, 1], counts)]
    tokens = rng.integers(6, size=22)  # few, so that they come again
    dec, cache = make(weights, 3, 24, 4, 24, 4, 16)
    rep, pres, freq = np.float32([1.25, 2, 1.5]), np.float32([0.5, 1, -0.25]), np.float32([0.25, -0.5, 2])
    kw = dict(given=None if given is None else i32(given))
    args = i32(tokens), i32(np.concatenate(trees)), i32(counts)
    dec.draft(*args, **kw)
    plain = dec.logits[:22].cpu().numpy().copy()
    cache.resize(i32([0, 0, 0]))
    rules = dict(zip(("repetition", "presence", "frequency"), (torch.from_numpy(x).cuda() for x in (rep, pres, freq))))
    if prompt_nodes is not None:
        rules["prompt_nodes"] = i32(prompt_nodes)
    dec.draft(*args, **kw, rules=rules)
    got, starts = dec.logits[:22].cpu().numpy(), np.concatenate([[0], np.cumsum(counts)])
    for b, tree in enumerate(trees):
        ids = tokens[starts[b]:starts[b + 1]].tolist()
        for i in range(len(tree)):
            prompt, said = ids[:asked[b]], [ids[j] for j in way(tree, i) if j >= asked[b]]
            want = plain[starts[b] + i].copy()
            for t in set(prompt + said):
                z, c = want[t], np.float32(said.count(t))
                z = z / rep[b] if z > 0 else z * rep[b]
                want[t] = z - freq[b] * c - (pres[b] if c else np.float32(0))
            np.testing.assert_array_equal(got[starts[b] + i], want)
            assert int(dec.tokens[starts[b] + i]) == int(want.argmax())
    no_device_error()


# -------------------------------------------------------------- attention ----
def test_trees_of_many_nodes_behind_wide_tables(cuda):
    """65 trees of 64 under tables of a million positions: what the tables could hold counts by tiles of 128 rows
    and the keys of a unit, and the answer is that of tables as wide as the requests are long."""
    batch = TreeBatch(20, [64 + 3 * b for b in range(65)], [64] * 65, 64, 8, 64, "bf16", 16)
    out, lse = batch.run()
    batch.table = np.concatenate([batch.table, np.full((65, 65536 - batch.table.shape[1]), -1)], 1)
    wide, lse_wide = batch.run()
    assert torch.equal(wide, out) and torch.equal(lse_wide, lse)
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


def test_refused_rules_change_nothing(cuda, model):  # noqa: F811
    """A step whose rules are refused shortens no request that its targets would shorten, and moves no page."""
    from edgeexpert_b200._lib import TFError
    weights, _ = model
    dec, cache = make(weights, 3, 24, 6, 24, 4, 8)
    ids, parents = i32(np.arange(20)), i32([-1, 0, 0, 2, 1] * 4)
    dec.draft(ids[:15], parents[:15], i32([5, 5, 5]), given=i32([5, 5, 5]))

    def state():
        torch.cuda.synchronize()
        return [t.clone() for t in (cache.seq_lens, cache.page_table, cache.free_ring, cache.free_state)]

    before = state()
    assert before[0].tolist() == [5, 5, 5]
    f, words = torch.ones(3, device="cuda"), -(-VOCAB // 32)
    bits = i32(np.full((5, words), -1))
    for bad in (dict(repetition=f[:2]), dict(presence=f.double()), dict(frequency=f.cpu()), dict(temperature=1.0),
                dict(history=i32(np.zeros((3, 4)))), dict(history=i32(np.zeros((1, 4))).expand(3, 4), history_lens=i32([4] * 3)),
                dict(history=i32(np.zeros(3)), history_lens=i32([0] * 3)), dict(allowed=bits[:1].expand(5, words)),
                dict(allowed=bits[:, :-1]), dict(allowed=bits[:4]), dict(allowed=bits, allowed_rows=i32([0])),
                dict(bias_tokens=i32([1])), dict(prompt_nodes=i32([1])), dict(prompt_nodes=f), dict(tokens=ids),
                dict(bias_starts=i32([0, 0, 0, 1]), bias_tokens=i32([1]), bias_values=f[:0])):
        with pytest.raises((TFError, TypeError)):
            dec.draft(ids[:5], parents[:5], i32([2, 10, 0]), rules=bad)
        assert all(torch.equal(a, b) for a, b in zip(before, state())), bad
    dec.draft(ids[:5], parents[:5], i32([2, 10, 0]), rules=dict(allowed=bits, repetition=f))
    assert cache.seq_lens.tolist()[0] == 2 and cache.seq_lens.tolist()[1] >= 6 and cache.seq_lens.tolist()[2] == 0
    no_device_error()


def test_a_step_by_another_stream(cuda, model):  # noqa: F811
    """Prompts, trees, masks and penalties on a stream of their own, with the other stream busy: the same bits."""
    weights, _ = model
    rng = np.random.default_rng(12)
    r = Round(rng, [rng.integers(VOCAB, size=n) for n in (4, 1, 6)], (5, 9, 0))
    bits, rows = r.masks()
    f = [torch.tensor(x, device="cuda") for x in ([1.5, 2.0, 1.25], [0.5, 0.25, 1.0], [0.25, 0.5, 0.125])]
    given, answers = i32([len(k) for k in r.known]), []
    rules = dict(allowed=torch.from_numpy(bits).cuda(), allowed_rows=i32(rows), repetition=f[0], presence=f[1], frequency=f[2])
    args = i32(np.concatenate(r.tokens)), i32(np.concatenate(r.trees)), i32([len(t) for t in r.tokens])
    for stream in (None, torch.cuda.Stream()):
        dec, cache = make(weights, 3, 24, 6, 32, 4, 16)
        noise = torch.randn(2000, 2000, device="cuda")
        torch.cuda.synchronize()
        if stream is not None:
            for _ in range(20):
                noise = noise @ noise / 50
        dec.draft(*args, given=given, rules=rules, stream=stream)
        torch.cuda.synchronize()
        n = sum(map(len, r.tokens))
        answers.append([x.clone() for x in (dec.counts, dec.new_tokens, dec.logits[:n], cache.seq_lens, cache.k, cache.v)])
    assert all(torch.equal(a, b) for a, b in zip(*answers))
    for b in range(3):
        path, fresh = r.expected(b)
        assert answers[0][0].tolist()[b] == len(path) and answers[0][1][b, :len(fresh)].tolist() == fresh
    no_device_error()
