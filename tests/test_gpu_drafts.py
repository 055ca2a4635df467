"""GPU tests of the drafted trees of a ragged batch (positions and ancestors,
attention, acceptance) against plain implementations in 64 bits.

Tolerances: whole numbers and moved values are equal; attention's are those of
the ragged batch (test_gpu_paged.py), its arithmetic being the same: with u the
unit roundoff of the 16-bit type, e = 2^-24 and A = sum p|v| / sum p, u A for the
weights' rounding and u A for the result's, 2 s A for scores off by s = (dim + 16)
e max(sum |q k|) scale, and keys * 2^-25 max|v| for weights below fp16's normal
range; lse: s, a rounding for each addition of the sum, and its own."""
import numpy as np
import pytest
import torch
from test_gpu_paged import DT, E32, U, Batch, f64, i32, no_device_error

pytestmark = pytest.mark.gpu


def random_parents(rng, n, roots=1):
    """Every node under any of those before it; the first `roots` are roots."""
    return np.array([-1 if i < roots else int(rng.integers(i)) for i in range(n)], dtype=np.int64)


def way(parents, i):
    """The nodes from the root to i."""
    found = [i]
    while parents[found[-1]] >= 0:
        found.append(int(parents[found[-1]]))
    return found[::-1]


def masks_of(trees):
    """Truth values [n][n] of each tree: node j is on the way to node i."""
    masks = []
    for parents in trees:
        m = np.zeros((len(parents), len(parents)), bool)
        for i in range(len(parents)):
            m[i, way(parents, i)] = True
        masks.append(m)
    return masks


def words_of(masks, words, padding=0):
    """int32 [T][words] as the operators read them."""
    rows = []
    for m in masks:
        full = np.zeros((len(m), words * 32), np.uint64)
        full[:, :m.shape[1]] = m
        rows.append((full.reshape(len(m), words, 32) << np.arange(32, dtype=np.uint64)).sum(-1))
    rows.append(np.zeros((padding, words), np.uint64))
    return torch.from_numpy(np.concatenate(rows).astype(np.uint32).view(np.int32)).cuda()


def flags():
    """The context's device error, which reading clears."""
    from edgeexpert_b200._lib import Context, TFError
    try:
        return Context.get(torch.cuda.current_device()).check_device() != 0
    except TFError:
        return True


# ------------------------------------------------------------------- plan ----
PLANS = [([1], 1), ([12], 12), ([0, 5, 0, 32, 1], 32), ([33, 2, 64], 64), ([3], 64), ([65, 128, 1], 128),
         ([256, 17, 200], 256), ([1] * 300, 1), ([2, 0] * 90, 40), ([0], 3)]


def plan(trees, lens, most, base=0, words=None, padding=0, first=0, parents=None, stream=None):
    from edgeexpert_b200.drafts import DraftTree
    counts = [len(t) for t in trees]
    words = -(-most // 32) if words is None else words
    T = first + sum(counts) + padding
    starts = first + np.concatenate([[0], np.cumsum(counts)])
    if parents is None:
        parents = np.concatenate([np.full(first, 5), *trees, np.full(padding, 7)])
    positions, ancestors = i32(np.full(T, 9)), i32(np.full((T, words), 9))
    DraftTree().encode_plan(i32(parents), i32(lens), i32(starts), positions, ancestors, most, position_base=base,
                            stream=stream)
    torch.cuda.synchronize()
    return positions.cpu().numpy(), ancestors.cpu().numpy().view(np.uint32), starts


def assert_plan(answer, trees, lens, base):
    positions, ancestors, starts = answer
    words = ancestors.shape[1]
    for tree, length, a in zip(trees, lens, starts):
        for i in range(len(tree)):
            w = way(tree, i)
            assert positions[a + i] == base + length - len(tree) + len(w) - 1
            bits = sum(1 << x for x in w)
            assert [int(x) for x in ancestors[a + i]] == [bits >> (32 * k) & 0xFFFFFFFF for k in range(words)]
    outside = np.r_[0:starts[0], starts[-1]:len(positions)]
    assert (positions[outside] == -1).all() and (ancestors[outside] == 0).all()


@pytest.mark.parametrize("counts,most", PLANS)
def test_plan(cuda, counts, most):
    rng = np.random.default_rng(most)
    for roots, words, padding, first in ((1, None, 0, 0), (2, 9, 5, 3), (1, None, 300, 0)):
        trees = [random_parents(rng, n, roots) for n in counts]
        lens = [n + int(rng.integers(5000)) for n in counts]
        assert_plan(plan(trees, lens, most, base=41, words=words, padding=padding, first=first), trees, lens, 41)
    no_device_error()


@pytest.mark.parametrize("n", [31, 32, 33, 255, 256])
def test_plan_of_chains_and_stars(cuda, n):
    """The deepest tree and the flattest."""
    trees = [np.arange(n) - 1, np.minimum(np.arange(n) - 1, 0)]
    assert_plan(plan(trees, [n + 3, n], 256), trees, [n + 3, n], 0)


def test_plan_of_bad_trees(cuda):
    """Parents that are not earlier nodes count as roots, nodes beyond the bound are left out; both are reported."""
    tree = np.array([-1, 0, 2, 7, 1, -5, 4])
    mended = np.array([-1, 0, -1, -1, 1, -1, 4])
    assert_plan(plan([tree], [10], 7), [mended], [10], 0)
    assert flags()
    positions, ancestors, _ = plan([np.arange(6) - 1, np.array([-1])], [8, 2], 4)
    assert positions.tolist() == [2, 3, 4, 5, -1, -1, 1] and ancestors[:, 0].tolist() == [1, 3, 7, 15, 0, 0, 1]
    assert flags()
    no_device_error()


# -------------------------------------------------------------- attention ----
def tree_reference(q, keys, values, past, mask, at, scale, window):
    """One request: keys / values [positions][nkv][hd], the last of them its nodes; node i sees the keys
    below `past` (with a window those above at[i] - window) and the nodes of mask[i]."""
    n, nq, hd = q.shape
    nkv = keys.shape[1]
    out, lse, A = np.zeros((n, nq, hd)), np.full((n, nq), -np.inf), np.zeros((n, nq, hd))
    most = 0.0
    for i in range(n):
        lo = max(0, max(at[i], past) - window + 1) if window else 0
        seen = np.r_[min(lo, past):past, past + np.flatnonzero(mask[i][:len(keys) - past])].astype(np.int64)
        if not len(seen):
            continue
        for h in range(nq):
            k, v = keys[seen, h * nkv // nq], values[seen, h * nkv // nq]
            s = (k @ q[i, h]) * scale
            most = max(most, float((np.abs(k) @ np.abs(q[i, h])).max()) * scale)
            w = np.exp(s - s.max())
            out[i, h], A[i, h] = (w @ v) / w.sum(), (w @ np.abs(v)) / w.sum()
            lse[i, h] = s.max() + np.log(w.sum())
    return out, lse, A, (hd + 16) * E32 * most


class TreeBatch(Batch):
    """A batch whose query tokens are nodes; `masks` any truth values (None: random trees')."""

    def __init__(self, *args, masks=None, words=None, **kw):
        super().__init__(*args, **kw)
        rng = np.random.default_rng(kw.get("seed", 0) + 99)
        self.trees = [random_parents(rng, n) for n in self.counts]
        self.masks = masks_of(self.trees) if masks is None else masks
        most = max([1] + self.counts)
        self.words = -(-most // 32) if words is None else words
        past = [self.P + max(0, length - n) for length, n in zip(self.lens, self.counts)]
        self.at = [p + m.sum(1) - 1 for p, m in zip(past, self.masks)]
        self.padding = len(self.q) - int(self.starts[-1])
        self.ancestors = words_of(self.masks, self.words, self.padding)
        self.positions = i32(np.concatenate([*self.at, np.full(self.padding, -1)]))

    def run(self, window=0, max_query=None, stream=None, out=None, lse=True, q=None):
        from edgeexpert_b200.drafts import TreeAttention
        from edgeexpert_b200.paged import PagedKV
        op, kv = TreeAttention(), PagedKV(self.k, self.v)
        q = self.q if q is None else q
        T, nq, hd = q.shape
        mq = max(1, max(self.counts)) if max_query is None else max_query
        out = torch.full((T, nq, hd), 7.0, dtype=self.dt, device="cuda") if out is None else out
        lse = torch.full((T, nq), 7.0, device="cuda") if lse else None
        args = (i32(self.table), i32(self.lens), i32(self.starts))
        prefix = i32(self.prefix_pages) if self.P else None
        answers = []
        for left in (255, 66):  # a workspace of arbitrary contents: NaN, and numbers
            ws = torch.full((op.workspace_bytes(kv, nq, T, len(self.lens), self.P, mq),), left, dtype=torch.uint8,
                            device="cuda")
            torch.cuda.synchronize()
            op.encode(q, kv, *args, self.ancestors, out, ws, prefix_pages=prefix, prefix_len=self.P, max_query=mq,
                      scale=self.scale, window=window, positions=self.positions if window else None, lse=lse,
                      stream=stream)
            torch.cuda.synchronize()
            answers.append(out.clone())
        assert torch.equal(answers[0].view(torch.int16), answers[1].view(torch.int16))
        return out, lse

    def reference(self, b, window):
        own, shared = f64(self.both[1 + b]), f64(self.both[0])
        keys, values = (np.concatenate([shared[i], own[i]]) for i in (0, 1))
        t = slice(self.starts[b], self.starts[b + 1])
        past = self.P + self.lens[b] - self.counts[b]
        mask = self.masks[b]
        if past < self.P:  # more nodes than positions: the first ones have none
            mask, past = mask[:, self.P - past:], self.P
        return (t, keys, values) + tree_reference(f64(self.q[t]), keys, values, past, mask, self.at[b], self.scale, window)

    def check(self, out, lse, window=0):
        out, lse, u = f64(out), f64(lse), U[self.dt]
        for b in range(len(self.lens)):
            t, keys, values, ro, rl, A, s = self.reference(b, window)
            seen, N = np.isfinite(rl), len(keys)
            small = N * 2.0 ** -25 * (np.abs(values).max() if N else 0) if self.dt == torch.float16 else 0
            tol = (2 * u + 2 * s + 16 * E32) * A + small + 2.0 ** -25
            assert (np.abs(out[t] - ro) <= tol).all(), (b, np.abs(out[t] - ro).max())
            assert (lse[t][~seen] == -np.inf).all() and (out[t][~seen] == 0).all()
            err = np.abs(lse[t][seen] - rl[seen])
            assert (err <= s + N * E32 + 4 * E32 * np.abs(rl[seen]) + 4 * E32).all(), (b, err.max())
        assert (out[self.starts[-1]:] == 0).all() and (lse[self.starts[-1]:] == -np.inf).all()


TREES = [
    # prefix, lens (nodes among them), nodes, nq, nkv, hd, dtype, page, window
    (0, [1], [1], 16, 8, 256, "fp16", 16, 0),
    (0, [712], [12], 16, 8, 256, "fp16", 16, 0),
    (0, [30, 4, 700, 64], [16, 4, 16, 3], 16, 8, 256, "fp16", 16, 0),
    (0, [64, 65, 300, 63], [64, 64, 64, 63], 16, 8, 256, "fp16", 64, 0),        # a tree and no history; ends of tiles
    (317, [17, 40], [9, 1], 16, 8, 256, "fp16", 16, 0),
    (513, [60, 131, 20], [20, 40, 20], 16, 4, 128, "bf16", 32, 0),
    (130, [9, 0, 31, 8], [1, 0, 4, 8], 16, 2, 64, "bf16", 17, 0),               # a request without a turn
    (501, [1500, 3, 800], [5, 3, 1], 16, 2, 64, "bf16", 16, 640),               # windows that leave the prefix, and reach it
    (400, [150, 200, 103], [100, 90, 3], 12, 4, 256, "bf16", 24, 128),
    (0, [900, 450], [33, 32], 4, 4, 128, "fp16", 8, 100),
    (0, [260, 300], [256, 200], 16, 8, 256, "fp16", 16, 0),                      # the largest trees: several row tiles
    (77, [300], [256], 8, 1, 128, "bf16", 48, 0),
    (300, [20, 45], [2, 33], 4, 4, 80, "fp16", 16, 0),                           # odd head sizes
    (77, [12], [5], 3, 1, 24, "bf16", 8, 0),
    (129, [40, 33], [7, 33], 4, 4, 512, "fp16", 16, 0),
    (260, [17, 30], [1, 3], 40, 1, 64, "bf16", 16, 0),                           # 40 heads to one KV head
    (64, [70] * 40, [6] * 40, 16, 8, 256, "fp16", 16, 0),
    (900, [50 + 3 * i for i in range(70)], [1 + i % 13 for i in range(70)], 16, 2, 128, "bf16", 16, 0),
    (0, [5000, 100, 9000], [60, 60, 60], 16, 8, 128, "fp16", 32, 0),
]


@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree_attention(cuda, case):
    prefix, lens, counts, nq, nkv, hd, dtype, page, window = TREES[case]
    batch = TreeBatch(prefix, lens, counts, nq, nkv, hd, dtype, page, seed=case, by_head=case % 3 == 1, padding=case % 4)
    batch.check(*batch.run(window), window)
    no_device_error()


@pytest.mark.parametrize("counts,prefix,nq,nkv,hd", [([7, 3], 0, 8, 8, 64), ([40, 5, 64], 0, 16, 4, 128),
                                                     ([100, 33], 200, 16, 8, 256), ([9, 2], 50, 4, 4, 512)])
def test_any_bits_are_taken(cuda, counts, prefix, nq, nkv, hd):
    """Masks that are no tree's: random ones, later nodes among them, bits beyond the nodes, and rows without
    any, which see nothing where there is no history either."""
    rng = np.random.default_rng(5)
    words = -(-max(counts) // 32) + 1
    masks = []
    for n in counts:
        m = rng.random((n, words * 32)) < 0.3
        m[n // 2] = False
        masks.append(m)
    lens = [counts[0]] + [n + 20 for n in counts[1:]]  # the first has no history
    batch = TreeBatch(prefix, lens, counts, nq, nkv, hd, "fp16", 16, seed=6, masks=masks, words=words, padding=1)
    out, lse = batch.run()
    batch.masks = [m[:, :n] for m, n in zip(masks, counts)]
    batch.check(out, lse)
    if not prefix:
        assert (lse[counts[0] // 2] == -np.inf).all()


def test_more_nodes_than_positions(cuda):
    """Lengths that do not hold all nodes: nodes without a position are nobody's key."""
    batch = TreeBatch(64, [3, 1, 2], [5, 1, 2], 8, 1, 128, "fp16", 1)
    batch.check(*batch.run())


@pytest.mark.parametrize("counts,hd", [([6, 3], 256), ([40, 9], 128), ([3, 5], 64), ([3, 2], 512)])
def test_nodes_that_others_see(cuda, counts, hd):
    """Infinities and NaN in a node's key and value: only the nodes below it see them."""
    lens = [c + 13 + 5 * i for i, c in enumerate(counts)]
    trees = [np.minimum(np.arange(n) - 1, 1) for n in counts]  # 0 - 1 - {2, 3, ...}
    batch = TreeBatch(40, lens, counts, 8, 4, hd, "fp16", 16, seed=11, masks=masks_of(trees))
    at = lens[0] - 1  # the last node of the first tree
    page, place = int(batch.table[0, at // 16]), at % 16
    batch.v[page, place, :, 0] = float("inf")
    batch.v[page, place, 0, 1] = float("nan")
    batch.k[page, place, 1, 0] = float("nan")
    out, lse = (f64(x) for x in batch.run())
    for b, n in enumerate(counts):
        t, _, _, ro, _, A, s = batch.reference(b, 0)
        hit = np.arange(n) == n - 1 if b == 0 else np.zeros(n, bool)
        assert (np.abs(out[t] - ro)[~hit] <= ((2 * U[torch.float16] + 2 * s + 16 * E32) * A + 1e-4)[~hit]).all()
        assert not np.isfinite(out[t][hit][..., 0]).any() and not np.isfinite(lse[t][hit][:, 2:4]).any()


@pytest.mark.parametrize("counts,hd", [([6, 3], 256), ([40, 9], 128), ([3, 5], 64), ([3, 2], 512)])
def test_windows_that_have_left_the_history(cuda, counts, hd):
    """Positions far ahead of the history: the nodes alone are seen, also by rows that are computed by
    themselves because a node beside them is infinite."""
    lens = [c + 13 + 5 * i for i, c in enumerate(counts)]
    trees = [np.minimum(np.arange(n) - 1, 1) for n in counts]  # 0 - 1 - {2, 3, ...}
    batch = TreeBatch(40, lens, counts, 8, 4, hd, "fp16", 16, seed=12, masks=masks_of(trees))
    batch.at = [a + 5000 for a in batch.at]
    batch.positions = i32(np.concatenate(batch.at))
    batch.check(*batch.run(window=64), window=64)
    at = lens[0] - 1  # the last node of the first tree
    batch.v[int(batch.table[0, at // 16]), at % 16] = float("inf")
    out, _ = batch.run(window=64)
    for b, n in enumerate(counts):
        t, _, _, ro, _, A, s = batch.reference(b, 64)
        fine = np.arange(n) != (n - 1 if b == 0 else -1)
        assert (np.abs(f64(out)[t] - ro)[fine] <= ((2 * U[torch.float16] + 2 * s + 16 * E32) * A + 1e-4)[fine]).all()
    no_device_error()


def test_chains_are_the_causal_batch(cuda):
    """A chain's ancestors are all nodes before it: the ragged batch's causal attention."""
    counts = [5, 1, 3]
    chains = [np.tril(np.ones((n, n), bool)) for n in counts]
    batch = TreeBatch(200, [60, 7, 41], counts, 16, 8, 256, "fp16", 16, seed=2, masks=chains)
    out, lse = batch.run()
    causal = Batch(200, [60, 7, 41], counts, 16, 8, 256, "fp16", 16, seed=2)
    assert torch.equal(causal.q, batch.q)
    causal.check(out, lse)


def test_tree_attention_by_another_stream_strides_and_repeats(cuda):
    batch = TreeBatch(700, [90, 5, 300], [40, 1, 30], 16, 4, 128, "fp16", 16, seed=8)
    ref, _ = batch.run()
    T = len(batch.q)
    wide = torch.zeros(T, 24 * 128, dtype=torch.float16, device="cuda")
    wide[:, 256:256 + 2048] = batch.q.flatten(1)
    out = torch.zeros(T, 20 * 128, dtype=torch.float16, device="cuda")
    for _ in range(3):
        got, _ = batch.run(stream=torch.cuda.Stream(), lse=False, q=wide[:, 256:256 + 2048].unflatten(1, (16, 128)),
                           out=out[:, 512:512 + 2048].unflatten(1, (16, 128)))
        assert torch.equal(got, ref)
    assert (out[:, :512] == 0).all() and (out[:, 512 + 2048:] == 0).all()


def test_tree_attention_with_a_loose_bound(cuda):
    batch = TreeBatch(150, [90, 40, 7], [30, 1, 3], 16, 4, 128, "bf16", 16, seed=21, words=8)
    for bound in (30, 64, 256, 2 ** 31 - 1):  # (no request has more than there are tokens)
        batch.check(*batch.run(max_query=bound))
    no_device_error()


def test_tree_attention_in_a_graph(cuda):
    """Captured once, replayed with other lengths and trees."""
    from edgeexpert_b200.drafts import TreeAttention
    from edgeexpert_b200.paged import PagedKV
    batch = TreeBatch(200, [100, 100], [20, 12], 16, 8, 256, "fp16", 16, seed=4)
    op, kv = TreeAttention(), PagedKV(batch.k, batch.v)
    ws = torch.empty(op.workspace_bytes(kv, 16, 32, 2, 200, 20), dtype=torch.uint8, device="cuda")
    table, lens, starts, pages = i32(batch.table), i32([100, 100]), i32(batch.starts), i32(batch.prefix_pages)
    out, lse = torch.zeros_like(batch.q), torch.zeros(32, 16, device="cuda")

    def call():
        op.encode(batch.q, kv, table, lens, starts, batch.ancestors, out, ws, prefix_pages=pages, prefix_len=200,
                  max_query=20, lse=lse)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = np.random.default_rng(1)
    for now in ([100, 100], [21, 77], [30, 12]):
        lens.copy_(i32(now))
        batch.masks = masks_of([random_parents(rng, n) for n in batch.counts])
        batch.ancestors.copy_(words_of(batch.masks, batch.words))
        graph.replay()
        torch.cuda.synchronize()
        batch.lens = now
        keep, batch.both = batch.both, [batch.both[0]] + [x[:, :n] for x, n in zip(batch.both[1:], now)]
        batch.check(out, lse)
        batch.both = keep


def test_tree_attention_calls_at_once(cuda):
    """Two batches on two streams at the same time, each with a workspace of its own; nothing waits between."""
    from edgeexpert_b200.drafts import TreeAttention
    from edgeexpert_b200.paged import PagedKV
    op, calls = TreeAttention(), []
    for spec in ((513, [60, 131, 20, 900], [20, 40, 20, 1], 16, 4, 128, "bf16", 32), (0, [700, 30], [12, 9], 16, 8, 256, "fp16", 16)):
        x = TreeBatch(*spec, seed=len(calls))
        want, _ = x.run()
        kv, mq, T, nq = PagedKV(x.k, x.v), max(x.counts), len(x.q), x.q.shape[1]
        ws = torch.empty(op.workspace_bytes(kv, nq, T, len(x.lens), x.P, mq), dtype=torch.uint8, device="cuda")
        prefix = i32(x.prefix_pages) if x.P else None
        args = (x.q, kv, i32(x.table), i32(x.lens), i32(x.starts), x.ancestors)
        calls.append((x, want, args, ws, prefix, mq, torch.cuda.Stream(), [torch.full_like(x.q, 7.0) for _ in range(20)]))
    torch.cuda.synchronize()
    for i in range(20):
        for x, _, args, ws, prefix, mq, stream, outs in calls:
            op.encode(*args, outs[i], ws, prefix_pages=prefix, prefix_len=x.P, max_query=mq, scale=x.scale, stream=stream)
    torch.cuda.synchronize()
    for _, want, *_, outs in calls:
        assert all(torch.equal(out, want) for out in outs)
    no_device_error()


def test_no_tokens(cuda):
    """A step in which nobody has a token: every operator takes it and writes what it has to."""
    from edgeexpert_b200.drafts import DraftAccept, DraftTree, TreeAttention
    from edgeexpert_b200.paged import PagedKV
    none, starts, lens = i32([]), i32([0, 0, 0]), i32([5, 0])
    DraftTree().encode_plan(none, lens, starts, none.clone(), i32(np.zeros((0, 1))), 4)
    k = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device="cuda")
    op, kv, q = TreeAttention(), PagedKV(k, k.clone()), torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    ws = torch.empty(max(16, op.workspace_bytes(kv, 4, 0, 2, 0, 4)), dtype=torch.uint8, device="cuda")
    op.encode(q, kv, i32([[0], [-1]]), lens, starts, i32(np.zeros((0, 1))), q.clone(), ws, max_query=4)
    counts, targets, paths, tokens = i32([7, 7]), i32([7, 7]), i32(np.full((2, 4), 7)), i32(np.full((2, 4), 7))
    DraftAccept().encode(none, none, none, lens, starts, counts, paths, tokens, targets, max_query=4)
    torch.cuda.synchronize()
    assert counts.tolist() == [0, 0] and targets.tolist() == [-1, -1]
    assert (paths == -1).all() and (tokens == -1).all()
    no_device_error()


def test_tree_attention_refusals(cuda):
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.drafts import TreeAttention
    from edgeexpert_b200.paged import PagedKV
    batch = TreeBatch(40, [20, 30], [3, 2], 8, 4, 64, "fp16", 16)
    op, kv = TreeAttention(), PagedKV(batch.k, batch.v)
    out = torch.zeros_like(batch.q)
    ws = torch.empty(op.workspace_bytes(kv, 8, 5, 2, 40, 3), dtype=torch.uint8, device="cuda")

    def call(q=batch.q, table=None, lens=None, starts=None, bits=batch.ancestors, out=out, ws=ws, **kw):
        kw = dict(dict(prefix_pages=i32(batch.prefix_pages), prefix_len=40, max_query=3), **kw)
        op.encode(q, kv, i32(batch.table) if table is None else table, i32([20, 30]) if lens is None else lens,
                  i32([0, 3, 5]) if starts is None else starts, bits, out, ws, **kw)

    call()
    call(window=3, positions=batch.positions)
    for bad in (dict(q=batch.q.bfloat16()), dict(scale=0.0), dict(scale=float("nan")), dict(max_query=0),
                dict(prefix_len=1000), dict(prefix_pages=None), dict(ws=ws[:0]), dict(starts=i32([0, 1])),
                dict(lens=torch.tensor([20, 30], device="cuda")), dict(table=i32(batch.table[:1])),
                dict(lse=torch.zeros(3, device="cuda")), dict(bits=batch.ancestors[:4]), dict(bits=batch.ancestors.long()),
                dict(bits=batch.ancestors[:, :0]), dict(bits=batch.ancestors[:, 0]), dict(window=2, positions=batch.positions),
                dict(window=64), dict(window=64, positions=batch.positions[:2]), dict(bits=batch.ancestors.cpu()),
                dict(out=out.cpu()), dict(positions=batch.positions.cpu()), dict(ws=ws.cpu())):
        with pytest.raises(TFError):
            call(**bad)
    no_device_error()
    # pages outside the pool and more nodes than announced are reported, not read
    for bad in (dict(table=i32(np.full_like(batch.table, 10 ** 6))), dict(prefix_pages=i32([-1, -1, -1])),
                dict(starts=i32([0, 5, 5]))):
        call(**bad)
        assert flags()
    no_device_error()


# ------------------------------------------------------------- acceptance ----
def walk(parents, drafted, choices, given):
    """One request: the kept nodes and the new tokens."""
    if not len(parents):
        return [], []
    given = min(max(given, 1), len(parents))
    path = list(range(given))
    while True:
        after = [i for i in range(given, len(parents)) if parents[i] == path[-1] and drafted[i] == choices[path[-1]]]
        if not after:
            return path, [int(choices[i]) for i in path[given - 1:]]
        path.append(after[0])


class Drafts:
    """Random trees whose choices follow one of their ways for a while, in pools of all layers."""

    def __init__(self, counts, lens, layers, nkv, hd, page, dtype="fp16", seed=0, vocab=5, given=None, by_head=False):
        rng = np.random.default_rng(seed)
        self.counts, self.lens, self.page = counts, lens, page
        self.trees = [random_parents(rng, n) for n in counts]
        self.given = [1] * len(counts) if given is None else given
        for tree, g in zip(self.trees, self.given):
            for i in range(1, min(g, len(tree))):
                tree[i] = i - 1
        # few different tokens: twins among children, choices that are met by chance
        self.drafted, self.choices = ([rng.integers(vocab, size=n) for n in counts] for _ in range(2))
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        held = [-(-n // page) for n in lens]
        total = sum(held) + 3
        ids, at = rng.permutation(total), 0
        self.table = np.full((len(lens), max(1, max(held))), -1)
        for b, h in enumerate(held):
            self.table[b, :h] = ids[at:at + h]
            at += h
        shape = (layers, total, nkv, page, hd) if by_head else (layers, total, page, nkv, hd)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.k, self.v = (torch.randn(shape, device="cuda", generator=gen).to(DT[dtype]) for _ in range(2))
        if by_head:
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)

    def run(self, most, op=None, stream=None, layers=True, given=True):
        from edgeexpert_b200.drafts import DraftAccept
        from edgeexpert_b200.paged import PagedKVLayers
        B = len(self.counts)
        self.out = [i32(np.full(s, 77)) for s in ((B,), (B, most), (B, most), (B,))]

        def flat(x):
            return i32(np.concatenate([*x, [3, 3]]))  # (two rows of padding)

        (op or DraftAccept()).encode(flat(self.drafted), flat(self.trees), flat(self.choices), i32(self.lens),
                                     i32(self.starts), *self.out, max_query=most, given=i32(self.given) if given else None,
                                     layers=PagedKVLayers(self.k, self.v) if layers else None,
                                     page_table=i32(self.table) if layers else None, stream=stream)
        torch.cuda.synchronize()
        return [x.cpu().numpy() for x in self.out]

    def expected(self, most):
        """What run answers, and the pools after it."""
        k, v = self.k.clone(), self.v.clone()
        B = len(self.counts)
        counts, targets = np.zeros(B, int), np.full(B, -1)
        paths, tokens = np.full((B, most), -1), np.full((B, most), -1)
        for b, n in enumerate(self.counts):
            path, new = walk(self.trees[b][:most], self.drafted[b], self.choices[b], self.given[b])
            counts[b], paths[b, :len(path)], tokens[b, :len(new)] = len(path), path, new
            history = self.lens[b] - n
            if path:
                targets[b] = history + len(path)
            for to, at in enumerate(path):
                if to != at:
                    (p0, i0), (p1, i1) = (divmod(history + x, self.page) for x in (at, to))
                    for x in (k, v):
                        x[:, self.table[b, p1], i1] = x[:, self.table[b, p0], i0].clone()
        return [counts, paths, tokens, targets], k, v


ACCEPT = [
    # nodes, lens, most, layers, nkv, hd, page, dtype, vocab, given, by_head
    ([12], [712], 12, 30, 8, 256, 16, "fp16", 2, None, False),
    ([1], [1], 1, 2, 8, 256, 16, "fp16", 2, None, False),
    ([0, 5, 0, 9], [0, 5, 3, 40], 9, 3, 4, 128, 16, "bf16", 2, None, True),
    ([24, 8, 16] * 10, [24, 100, 77] * 10, 24, 5, 2, 64, 8, "fp16", 2, None, False),
    ([64, 33, 2], [70, 1000, 90], 64, 2, 1, 80, 1, "bf16", 1, None, False),        # one token: the deepest way of all
    ([256, 200], [256, 300], 256, 1, 3, 24, 17, "fp16", 1, None, True),
    ([20, 9, 30, 4], [25, 9, 64, 80], 30, 4, 8, 64, 24, "fp16", 2, [10, 9, 1, 99], False),
    ([3, 3], [3, 3], 40, 2, 2, 8, 4, "bf16", 3, [0, -4], False),
]


@pytest.mark.parametrize("case", range(len(ACCEPT)))
@pytest.mark.parametrize("seed", range(4))
def test_accept(cuda, case, seed):
    counts, lens, most, layers, nkv, hd, page, dtype, vocab, given, by_head = ACCEPT[case]
    d = Drafts(counts, lens, layers, nkv, hd, page, dtype, seed=seed, vocab=vocab, given=given, by_head=by_head)
    answer, k, v = d.expected(most)
    got = d.run(most, given=given is not None)
    for g, a in zip(got, answer):
        assert np.array_equal(g, a)
    assert torch.equal(d.k, k) and torch.equal(d.v, v)
    no_device_error()


def test_accept_of_chains_in_place(cuda):
    """A chain that is kept whole moves nothing; without pools only the lists are written."""
    d = Drafts([6, 4], [10, 4], 2, 2, 64, 16, seed=1)
    for b, n in enumerate(d.counts):
        d.trees[b] = np.arange(n) - 1
        d.choices[b][:-1] = d.drafted[b][1:]
    for layers in (True, False):
        answer, k, v = d.expected(6)
        for g, a in zip(d.run(6, layers=layers), answer):
            assert np.array_equal(g, a)
        assert answer[0].tolist() == [6, 4] and torch.equal(d.k, k) and torch.equal(d.v, v)
    no_device_error()


@pytest.mark.parametrize("layer_stride,page_stride", [((1 << 32) + 8, 64 * 64), (16 * 64, 1 << 30)])
def test_accept_far_into_the_pools(cuda, layer_stride, page_stride):
    """Elements beyond 2^32 of the first: by the layers' distance and by the pages'."""
    d = Drafts([8, 5], [20, 5], 2, 2, 32, 16, seed=5, vocab=1)
    layers, pages = d.k.shape[:2]
    extent = (layers - 1) * layer_stride + (pages - 1) * page_stride + 16 * 64
    answer, k, v = d.expected(8)
    assert any(p >= 0 and p != i for path in answer[1] for i, p in enumerate(path))  # (something moves)
    near, far = (d.k, d.v), []
    for x in near:
        far.append(torch.empty(extent, dtype=x.dtype, device="cuda").as_strided(x.shape, (layer_stride, page_stride, 64, 32, 1)))
        far[-1].copy_(x)
    d.k, d.v = far
    for g, a in zip(d.run(8), answer):
        assert np.array_equal(g, a)
    assert torch.equal(d.k, k) and torch.equal(d.v, v)
    no_device_error()


def test_no_choice_ends_the_way(cuda):
    """A choice of -1 is no token, and meets no node, whatever was drafted."""
    d = Drafts([4], [4], 1, 2, 64, 4, seed=3, vocab=1)
    d.trees[0] = np.array([-1, 0, 1, 2])
    d.drafted[0] = np.array([0, 0, -1, 0])
    d.choices[0] = np.array([0, -1, 0, 0])
    counts, paths, tokens, targets = d.run(4)
    assert counts.tolist() == [2] and paths.tolist() == [[0, 1, -1, -1]] and tokens.tolist() == [[0, -1, -1, -1]]
    assert targets.tolist() == [2]
    no_device_error()


def test_accept_of_bad_trees_and_pages(cuda):
    """A parent that is not earlier is nobody's; nodes beyond the bound and pages outside the pool are
    reported, and what they hold is not moved."""
    d = Drafts([5], [5], 1, 2, 64, 4, seed=3, vocab=1)
    d.trees[0] = np.array([-1, 0, 4, 1, -3])
    answer, k, v = d.expected(5)
    assert answer[1].tolist() == [[0, 1, 3, -1, -1]]
    for g, a in zip(d.run(5), answer):
        assert np.array_equal(g, a)
    assert torch.equal(d.k, k) and flags()
    d = Drafts([8], [8], 2, 2, 64, 4, seed=3, vocab=1)
    answer, k, v = d.expected(5)  # (max_query 5: the last three nodes are not looked at)
    for g, a in zip(d.run(5), answer):
        assert np.array_equal(g, a)
    assert torch.equal(d.k, k) and flags()
    d = Drafts([8], [8], 2, 2, 64, 4, seed=9, vocab=1)
    d.trees[0] = np.array([-1, 0, 0, 0, 0, 0, 0, 2])
    d.drafted[0][1] = 7  # 0 - 2 - 7: from page 1 to place 2 of page 0, and within page 0
    before = d.k.clone()
    for pages in ([[10 ** 6, -1]], [[-1, 0]], [[int(d.table[0, 0]), 10 ** 6]]):
        d.k.copy_(before)
        keep, d.table = d.table, np.array(pages)
        got = d.run(8)
        assert got[1][0, :3].tolist() == [0, 2, 7] and got[3].tolist() == [3] and flags()
        if pages[0][0] != int(keep[0, 0]):
            assert torch.equal(d.k, before)
        else:
            moved = before.clone()
            moved[:, keep[0, 0], 1] = before[:, keep[0, 0], 2]
            assert torch.equal(d.k, moved)
        d.table = keep
    no_device_error()


def test_accept_refusals(cuda):
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.drafts import DraftAccept
    from edgeexpert_b200.paged import PagedKVLayers
    op = DraftAccept()
    pool = torch.zeros(2, 4, 4, 2, 64, dtype=torch.float16, device="cuda")
    layers = PagedKVLayers(pool, pool.clone())

    def call(ids=i32([1, 2, 3]), parents=i32([-1, 0, 1]), lens=i32([3]), counts=i32([0]), paths=i32([[0] * 3]),
             max_query=3, layers=layers, table=i32([[0]]), **kw):
        op.encode(ids, parents, i32([1, 2, 3]), lens, i32([0, 3]), counts, paths, i32([[0] * 3]), i32([0]),
                  max_query=max_query, layers=layers, page_table=table, **kw)

    call()
    big = i32([[0] * 257])
    for bad in (dict(parents=i32([-1, 0])), dict(counts=i32([0, 0])), dict(paths=i32([[0] * 4])), dict(table=None),
                dict(table=i32([[0], [0]])), dict(ids=torch.tensor([1, 2, 3], device="cuda")),
                dict(given=i32([1, 1])), dict(lens=torch.tensor([3], dtype=torch.int32)), dict(max_query=0),
                dict(table=i32([[0]]).cpu()), dict(table=i32(np.zeros((1, 0))))):
        with pytest.raises(TFError):
            call(**bad)
    with pytest.raises(TFError):
        op.encode(i32([1]), i32([-1]), i32([1]), i32([1]), i32([0, 1]), i32([0]), big, big.clone(), i32([0]), max_query=257)
    with pytest.raises(TFError):
        PagedKVLayers(pool[0], pool[0])
    with pytest.raises(TFError):
        call(layers=PagedKVLayers(pool[:1].expand(2, 4, 4, 2, 64), pool[:1].expand(2, 4, 4, 2, 64)))
    no_device_error()
