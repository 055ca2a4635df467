"""GPU tests of DraftDecoder: rounds of drafted trees behind a shared prefix, with
prompts, rules and requests that are refused, against the paged decoder on each
way's tokens as one prompt (which test_gpu_paged.py holds against the contiguous
one).

Both run the same products on as many rows and differ in the attention alone, by
less than 1e-3 of its result a layer (two roundings of 2^-11 and what the weights'
rounding gives): two layers, four times that for what the rest of a layer may make
of it, 8e-3 between them.  That holds while both choose the same experts: the
choice is not continuous, and where the last expert in and the first one out are as
near as the hidden states are to each other, either is right.  So every layer's
experts are kept for every token; a row is compared if all tokens on its way have
the same ones, and where they differ the two that changed places must be a near
tie: a router logit is a product of the state, off by 8e-3 of its norm, with a row
of weights, so both sides' logits are within 2 * 8e-3 |state| |weights|, which is
below 0.5 here (16 experts whose logits spread over a few units).  Masks that allow
one token choose the way through a tree, so that nothing hangs on how near two
logits are."""
import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_drafts import random_parents, walk, way
from test_gpu_paged import f64, i32, no_device_error

pytestmark = pytest.mark.gpu
VOCAB = 1000


@pytest.fixture(scope="module")
def model():
    """(weights, the last hidden state of a sequence)."""
    from edgeexpert_b200.decoder import DecoderConfig, synthetic_decoder
    from edgeexpert_b200.paged import PagedDecoder, PagedKVCache
    cfg = DecoderConfig(d=256, f=128, fs=128, num_experts=16, top_k=8, num_q_heads=4, num_kv_heads=2, head_dim=64,
                        vocab=VOCAB, layers=2, max_context=96)
    dev = torch.device("cuda", 0)
    weights = synthetic_decoder(cfg, dev, torch.Generator(device=dev).manual_seed(7))

    def alone(tokens, T):
        """The last hidden state, and every token's experts, in steps of T rows."""
        cache = PagedKVCache(cfg.layers, cfg.num_kv_heads, cfg.head_dim, 1, 12, 12, T, page_size=16)
        dec = PagedDecoder(weights, T, cache, max_query=T)
        seen, routes = record(dec), []
        for at in range(0, len(tokens), T):
            part = tokens[at:at + T]
            dec.step(i32(part), i32([at + len(part)]))
            routes += [routes_of(seen, i) for i in range(len(part))]
        return f64(dec.h)[len(part) - 1], routes

    return weights, alone


def record(dec):
    """The layers' experts and their weights in the step after, as tensors."""
    run, seen = dec._moe, []

    def moe(i, stream):
        run(i, stream)
        if i == 0:
            seen.clear()
        seen.append((dec.idx.clone(), dec.wts.clone()))

    dec._moe = moe
    return seen


def routes_of(seen, row):
    """A row's experts by layer: {expert: weight}."""
    return [dict(zip(idx[row].tolist(), wts[row].tolist())) for idx, wts in seen]


class Compared:
    """Rows that were compared, and those whose tokens met other experts."""

    def __init__(self):
        self.rows = self.others = 0

    def close(self, row, routes, want, want_routes):
        assert len(routes) == len(want_routes)
        for mine, theirs in zip(routes, want_routes):
            for a, b in zip(mine, theirs):
                if a.keys() == b.keys():
                    continue
                # of each side the least likely of those that the other has not, against an expert of both
                common = max(a.keys() & b.keys(), key=a.get)
                out = np.log([min(a[e] for e in a.keys() - b.keys()) / a[common],
                              min(b[e] for e in b.keys() - a.keys()) / b[common]])
                assert abs(out[0] - out[1]) < 0.5, (a, b)
                self.others += 1
                return
        error = float(O.rel_error(row.astype(np.float32), want.astype(np.float32)))
        assert error < 8e-3
        self.rows += 1


def make(weights, requests, pages, max_pages, T, page_size, max_query):
    from edgeexpert_b200.drafts import DraftDecoder
    from edgeexpert_b200.paged import PagedKVCache
    cfg = weights.cfg
    cache = PagedKVCache(cfg.layers, cfg.num_kv_heads, cfg.head_dim, requests, pages, max_pages, T, page_size=page_size)
    return DraftDecoder(weights, T, cache, max_query=max_query), cache


class Round:
    """Trees of a round: each user's known tokens, then nodes under the last of them; one way down each
    (some end at once) and the token behind it."""

    def __init__(self, rng, known, nodes):
        self.known, self.trees, self.tokens, self.want = known, [], [], []
        for tokens, n in zip(known, nodes):
            g = len(tokens)
            parents = np.concatenate([np.arange(g) - 1, [rng.integers(g - 1, g + i) for i in range(n)]]).astype(np.int64)
            self.trees.append(parents)
            self.tokens.append(np.concatenate([tokens, rng.integers(VOCAB, size=n)]).astype(np.int64))
            kept = [p for p in (way(parents, i) for i in range(g - 1, g + n)) if len(p) >= g]
            path = kept[rng.integers(len(kept))] if g else []
            self.want.append((path, int(rng.integers(VOCAB))))

    def masks(self):
        """allowed, allowed_rows: on the way, the next token alone; elsewhere no mask."""
        bits, rows = [], []
        for tokens, (path, last) in zip(self.tokens, self.want):
            after = dict(zip(path, [int(tokens[j]) for j in path[1:]] + [last]))
            for i in range(len(tokens)):
                rows.append(len(bits) if i in after else -1)
                if i in after:
                    word = np.zeros(-(-VOCAB // 32), np.uint32)
                    word[after[i] // 32] = 1 << (after[i] % 32)
                    bits.append(word)
        return np.array(bits).view(np.int32), rows

    def expected(self, b):
        """Kept nodes and new tokens: a child before the way's that has its token is kept in its place."""
        tokens, (path, last) = self.tokens[b], self.want[b]
        choices = np.full(len(tokens), -9)
        for i, j in zip(path, path[1:]):
            choices[i] = tokens[j]
        if path:
            choices[path[-1]] = last
        return walk(self.trees[b], tokens, choices, len(self.known[b]))


def padded(rows, T):
    return i32(np.concatenate([rows, np.full(T - len(rows), -1)]))


def play(dec, cache, r, lens, T, refused=(), **rules):
    """A round; the answer is checked.  Returns the hidden states and experts by request."""
    live = [b for b in range(len(lens)) if len(r.tokens[b])]
    granted = [b for b in live if b not in refused]
    targets = [lens[b] + len(r.tokens[b]) if b in live else -1 for b in range(len(lens))]
    bits, rows = Round.masks(r)
    keep = [x for b in live for x in ([True] * len(r.tokens[b]) if b in granted else [False] * len(r.tokens[b]))]
    rows = [x for x, k in zip(rows, keep) if k]  # (the step's rows are those of the granted requests)
    seen = record(dec)
    counts, new = dec.draft(i32(np.concatenate(r.tokens)[:T]), i32(np.concatenate(r.trees)[:T]), i32(targets),
                            given=i32([len(k) for k in r.known]),
                            rules=dict(allowed=torch.from_numpy(bits).cuda(), allowed_rows=padded(rows, T), **rules))
    del dec._moe
    torch.cuda.synchronize()
    h, counts, new, paths = f64(dec.h), counts.tolist(), new.cpu().numpy(), dec.paths.cpu().numpy()
    starts = dec.draft_starts.tolist()
    assert dec.draft_state.tolist()[2:] == [len(live) - len(granted), sum(len(r.tokens[b]) for b in granted)]
    states = {}
    for b in range(len(lens)):
        if b not in granted:
            assert counts[b] == 0 and (new[b] == -1).all()
            continue
        path, fresh = r.expected(b)
        assert counts[b] == len(path) and paths[b, :len(path)].tolist() == path
        assert new[b, :len(fresh)].tolist() == fresh and (new[b, len(fresh):] == -1).all()
        lens[b] += len(path)
        states[b] = [(h[t], routes_of(seen, t)) for t in range(starts[b], starts[b + 1])]
    assert cache.seq_lens.tolist() == lens
    return states


class Text:
    """What the users have said and kept so far, with the experts that it met."""

    def __init__(self, users, T, tokens=(), routes=()):
        self.T = T
        self.tokens, self.routes = [list(tokens) for _ in range(users)], [list(routes) for _ in range(users)]

    def check(self, compared, alone, r, b, states, i):
        """Node i of request b's tree, kept or not, against its own way."""
        down = way(r.trees[b], i)
        want, routes = alone(self.tokens[b] + [int(r.tokens[b][j]) for j in down], self.T)
        compared.close(states[b][i][0], self.routes[b] + [states[b][j][1] for j in down], want, routes)

    def keep(self, r, b, states):
        path, fresh = r.expected(b)
        self.tokens[b] += [int(r.tokens[b][i]) for i in path]
        self.routes[b] += [states[b][i][1] for i in path]
        return np.array(fresh[-1:])


def test_rounds_of_trees_agree_with_the_kept_tokens_decoded_alone(cuda, model):
    weights, alone = model
    rng = np.random.default_rng(5)
    T, most, page = 60, 24, 4
    dec, cache = make(weights, 3, 60, 12, T, page, most)
    prefix = rng.integers(VOCAB, size=13)
    seen = record(dec)
    dec.step(i32(prefix), i32([13, -1, -1]))  # (plain steps as before)
    text = Text(3, T, prefix, [routes_of(seen, t) for t in range(13)])
    del dec._moe
    cache.share(0, 13)
    held = cache.free_state.tolist()[1]
    lens, compared = [0, 0, 0], Compared()
    known = [rng.integers(VOCAB, size=n) for n in (5, 1, 9)]  # prompts
    for turn, nodes in enumerate([(6, 12, 0), (15, 3, 20), (0, 9, 8), (23, 1, 2)]):
        r = Round(rng, known, nodes)
        states = play(dec, cache, r, lens, T)
        for b in range(3):
            for i in range(0, len(r.tokens[b]), 1 if turn == 0 else 3):
                text.check(compared, alone, r, b, states, i)
            known[b] = text.keep(r, b, states)
        assert cache.free_state.tolist()[1] == held - sum(-(-n // page) for n in lens)
    # the cache goes on from the kept nodes: a plain token behind each
    more = rng.integers(VOCAB, size=3)
    seen = record(dec)
    dec.step(i32(more), i32([n + 1 for n in lens]))
    h = f64(dec.h)
    for b in range(3):
        want, routes = alone(text.tokens[b] + [int(more[b])], T)
        compared.close(h[b], text.routes[b] + [routes_of(seen, b)], want, routes)
    assert compared.rows > compared.others  # (a token that met others leaves out all rows behind it)
    no_device_error()


def test_a_request_that_is_refused_keeps_its_length(cuda, model):
    """The list holds 40 tokens: the third user's sixteen do not fit behind the others'."""
    weights, alone = model
    rng = np.random.default_rng(8)
    dec, cache = make(weights, 3, 40, 12, 40, 4, 16)
    lens, text, compared = [0, 0, 0], Text(3, 40), Compared()
    known = [rng.integers(VOCAB, size=n) for n in (4, 7, 2)]
    r = Round(rng, known, (6, 9, 5))
    states = play(dec, cache, r, lens, 40)
    known = [text.keep(r, b, states) for b in range(3)]
    r = Round(rng, known, (15, 15, 15))
    before = lens[2]
    states = play(dec, cache, r, lens, 40, refused=[2])
    assert lens[2] == before
    for b in range(2):
        for i in range(0, 16, 5):
            text.check(compared, alone, r, b, states, i)
        known[b] = text.keep(r, b, states)
    r = Round(rng, known, (2, 0, 3))  # and then it has its turn
    states = play(dec, cache, r, lens, 40)
    for b in range(3):
        text.check(compared, alone, r, b, states, len(r.tokens[b]) - 1)
    assert compared.rows > compared.others  # (a token that met others leaves out all rows behind it)
    no_device_error()


def test_penalties_count_the_way_down_a_tree(cuda, model):
    """Without a mask, a chain whose tokens are all the best one: the presence penalty of a node falls on
    the tokens of its own way, in the logits that the step leaves behind."""
    weights, _ = model
    dec, cache = make(weights, 1, 8, 4, 12, 4, 8)
    history = i32([[5, 6, 5, 0]])
    kw = dict(history=history, history_lens=i32([3]), prompt_lens=i32([1]), presence=torch.tensor([0.5], device="cuda"),
              frequency=torch.tensor([0.25], device="cuda"))
    ids, parents = [5, 9, 9, 7], [-1, 0, 1, 0]
    dec.draft(i32(ids), i32(parents), i32([4]))
    plain = dec.logits[:4].clone()
    cache.resize(i32([0]))
    dec.draft(i32(ids), i32(parents), i32([4]), rules=kw)
    for i in range(4):
        said = [6, 5] + [ids[j] for j in way(np.array(parents), i)]
        want = plain[i].clone()
        for token in set(said):
            want[token] = want[token] - torch.tensor(0.25 * said.count(token), device="cuda") - 0.5
        assert torch.equal(dec.logits[i], want)
        assert int(dec.tokens[i]) == int(want.argmax())
    no_device_error()


def test_a_round_in_a_graph(cuda, model):
    """Captured once, replayed on other trees from other lengths."""
    weights, _ = model
    rng = np.random.default_rng(2)
    dec, cache = make(weights, 2, 20, 8, 16, 4, 8)
    ids, parents, targets, given = (i32(np.zeros(n)) for n in (16, 16, 2, 2))
    bits, rows = torch.zeros(16, -(-VOCAB // 32), dtype=torch.int32, device="cuda"), i32(np.zeros(16))
    rules = dict(allowed=bits, allowed_rows=rows)

    def call():
        dec.draft(ids, parents, targets, given=given, rules=rules)

    targets.fill_(-1)
    call()  # (workspaces)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    lens = [0, 0]
    known = [rng.integers(VOCAB, size=n) for n in (4, 1)]
    for nodes in ((4, 7), (7, 2), (1, 5)):
        r = Round(rng, known, nodes)
        mask, at = r.masks()
        n = sum(map(len, r.tokens))
        for to, x in ((ids, np.concatenate(r.tokens)), (parents, np.concatenate(r.trees)), (rows, at)):
            to.copy_(padded(x, 16))
        bits[:len(mask)] = torch.from_numpy(mask).cuda()
        targets.copy_(i32([k + len(t) for k, t in zip(lens, r.tokens)]))
        given.copy_(i32([len(k) for k in r.known]))
        graph.replay()
        torch.cuda.synchronize()
        assert dec.draft_state.tolist()[3] == n
        for b in range(2):
            path, fresh = r.expected(b)
            assert dec.counts.tolist()[b] == len(path) and dec.new_tokens[b, :len(fresh)].tolist() == fresh
            lens[b] += len(path)
            known[b] = np.array(fresh[-1:])
        assert cache.seq_lens.tolist() == lens
    no_device_error()
    del graph


def test_a_captured_round_outlives_larger_ones(cuda, model):
    """A step with longer histories than a captured one's takes a workspace of its own: the captured step's
    stays where it is."""
    weights, _ = model
    dec, cache = make(weights, 1, 8, 4, 8, 4, 4)
    short, history = dict(history=i32([[5] * 8]), history_lens=i32([8])), i32([[6] * 3000])
    ids, parents, targets = i32([1, 2]), i32([-1, 0]), i32([2])
    dec.draft(ids, parents, targets, rules=short)
    cache.resize(i32([0]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec.draft(ids, parents, targets, rules=short)
    graph.replay()
    torch.cuda.synchronize()
    want, small = (dec.tokens[:2].tolist(), dec.logits[:2].clone()), dec.rules_workspace
    cache.resize(i32([0]))
    dec.draft(ids, parents, targets, rules=dict(history=history, history_lens=i32([3000])))
    assert dec.rules_workspace.data_ptr() != small.data_ptr() and any(w is small for w in dec._workspaces)
    del small
    for _ in range(3):
        torch.full((1 << 16,), 255, dtype=torch.uint8, device="cuda")
    cache.resize(i32([0]))
    graph.replay()
    torch.cuda.synchronize()
    assert dec.tokens[:2].tolist() == want[0] and torch.equal(dec.logits[:2], want[1])
    no_device_error()
    del graph


def test_refusals(cuda, model):
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.drafts import DraftDecoder
    weights, _ = model
    dec, cache = make(weights, 2, 8, 4, 8, 4, 4)
    ids, parents, targets = i32([1, 2, 3]), i32([-1, 0, -1]), i32([2, 1])
    for bad in ((ids.long(), parents, targets), (ids, parents[:2], targets), (ids, parents.long(), targets),
                (ids, parents, i32([2])), (i32(np.zeros(9)), i32(np.zeros(9)), targets), (ids, parents, targets.cpu()),
                (ids[None], parents, targets)):
        with pytest.raises(TFError):
            dec.draft(*bad)
    with pytest.raises(TFError):
        dec.draft(ids, parents, targets, given=i32([1]))
    with pytest.raises(TFError):
        DraftDecoder(weights, 8, cache, max_query=257)
    assert cache.seq_lens.tolist() == [0, 0]
    dec.draft(ids, parents, targets)
    kept, free = cache.seq_lens.tolist(), cache.free_state[1].item()
    for bad in (dict(repetition=torch.ones(3, device="cuda")), dict(temperature=1), dict(history=i32([[1], [2]])),
                dict(allowed=i32(np.zeros((1, 1)))), dict(tokens=ids)):  # found when the nodes are there
        with pytest.raises((TFError, TypeError)):
            dec.draft(ids, parents, cache.seq_lens + i32([2, 1]), rules=bad)
        assert cache.seq_lens.tolist() == kept and cache.free_state[1].item() == free
    dec.draft(ids[:0], parents[:0], i32([-1, -1]))  # nothing to do
    assert dec.counts.tolist() == [0, 0]
    no_device_error()
