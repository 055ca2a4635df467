"""GPU tests of the rules on logits (penalties, biases, grammar masks, the best
token) against their definition in 64 bits.

Tolerance of a logit: the rule's up to five fp32 steps (division or product,
frequency * count, two subtractions, the bias) round by at most 2^-24 of a value
each, and no value on the way is larger than M = the sum of the steps' magnitudes;
then one rounding to the logits' type, u |z| + its smallest step / 2.  The token
is that of the largest 64-bit value wherever no other comes within twice that
fp32 tolerance of it; the others may be chosen where they do."""
import numpy as np
import pytest
import torch
from test_gpu_drafts import flags, masks_of, random_parents, words_of
from test_gpu_paged import i32, no_device_error

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24
TYPES = {"fp32": (torch.float32, 2.0 ** -24, 2.0 ** -150), "fp16": (torch.float16, 2.0 ** -11, 2.0 ** -25),
         "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134)}


class Rows:
    """Rows of a ragged batch and random rules on them."""

    def __init__(self, counts, V, dtype, history=(0, 50), prompt=0.5, biases=0, grammar=None, trees=False, seed=0,
                 padding=0, factors=True, hot=0.5):
        rng = np.random.default_rng(seed)
        self.counts, self.V, self.dtype = counts, V, dtype
        B, T = len(counts), sum(counts) + padding
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.logits = (torch.randn(T, V, device="cuda", generator=gen) * 4).to(TYPES[dtype][0])
        self.lens = rng.integers(history[0], history[1] + 1, B)
        longest = max(1, history[1])

        def tokens(*shape):  # repeated ones, some of them outside the vocabulary
            t = (rng.random(shape) ** 4 * V).astype(np.int64)
            return np.where(rng.random(shape) < 0.05, rng.choice([-1, V, V + 7, 2 ** 31 - 1, -2 ** 31], shape), t)

        self.history = tokens(B, longest)
        self.prompt = (self.lens * prompt).astype(np.int64)
        self.rep, self.pres, self.freq = ((1 + rng.random(B)).astype(np.float32), rng.normal(size=B).astype(np.float32),
                                          rng.normal(size=B).astype(np.float32)) if factors else (None,) * 3
        self.bias = None
        if biases:
            n = rng.integers(0, biases + 1, B)
            self.bias = (np.concatenate([[0], np.cumsum(n)]), tokens(n.sum()), rng.normal(size=n.sum()).astype(np.float32))
            self.bias[2][rng.random(n.sum()) < 0.2] = -np.inf
        self.allowed = self.rows = None
        if grammar is not None:
            words = -(-V // 32) + 1
            self.allowed = rng.integers(0, 2 ** 32, (max(1, T // 2), words), dtype=np.uint64).astype(np.uint32)
            self.allowed &= rng.integers(0, 2 ** 32, self.allowed.shape, dtype=np.uint64).astype(np.uint32)
            self.rows = rng.integers(-1, len(self.allowed), T)
            if grammar == "nothing":
                self.allowed[:] = 0
            if grammar == "own":  # row t is under row t of the masks
                self.allowed, self.rows = np.resize(self.allowed, (T, words)), None
        self.drafted = self.masks = None
        if trees:
            self.drafted = tokens(T)
            self.masks = masks_of([random_parents(rng, n) for n in counts])

    def workspace(self, op, T):
        return op.workspace_bytes(T, self.V, len(self.counts), self.history.shape[1],
                                  0 if self.bias is None else len(self.bias[1]))

    def run(self, out=None, logits=None, tokens=True, max_query=None, stream=None, words=None):
        from edgeexpert_b200.sampling import LogitRules
        op = LogitRules()
        logits = self.logits if logits is None else logits
        T, V = logits.shape
        out = torch.full_like(logits, 7.0) if out is None else out
        chosen = i32(np.full(T, 77)) if tokens else None
        most = max([1] + self.counts) if max_query is None else max_query

        def f32(x):
            return None if x is None else torch.from_numpy(x).cuda()

        kw = dict(history=i32(self.history), history_lens=i32(self.lens), prompt_lens=i32(self.prompt))
        kw.update(repetition=f32(self.rep), presence=f32(self.pres), frequency=f32(self.freq))
        if self.bias is not None:
            kw.update(bias_starts=i32(self.bias[0]), bias_tokens=i32(self.bias[1]), bias_values=f32(self.bias[2]))
        if self.allowed is not None:
            kw.update(allowed=torch.from_numpy(self.allowed.view(np.int32)).cuda(),
                      allowed_rows=None if self.rows is None else i32(self.rows))
        if self.drafted is not None:
            padding = T - int(self.starts[-1])
            words = -(-max([1] + self.counts) // 32) if words is None else words
            kw.update(token_ids=i32(self.drafted), ancestors=words_of(self.masks, words, padding))
        for left in (0, 255):
            ws = torch.full((self.workspace(op, T),), left, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            op.encode(logits, out, i32(self.starts), ws, max_query=most, tokens=chosen, stream=stream,
                      **kw)
            torch.cuda.synchronize()
            if out.data_ptr() == logits.data_ptr():
                break
        return out, chosen

    def reference(self, t):
        """The row's logits in 64 bits, and the tolerance of each in fp32."""
        b = int(np.searchsorted(self.starts, t, side="right")) - 1
        V = self.V

        def count(x):
            return np.bincount(x[(x >= 0) & (x < V)], minlength=V)

        h, prompt = self.history[b, :self.lens[b]], self.prompt[b]
        said, asked = count(h[prompt:]), count(h[:prompt])
        if self.drafted is not None:
            way = np.flatnonzero(self.masks[b][t - self.starts[b]])
            said = said + count(self.drafted[self.starts[b] + way])
        one = np.float32(1)
        rep, pres, freq = (float(x[b]) if x is not None else float(d) for x, d in
                           ((self.rep, one), (self.pres, 0 * one), (self.freq, 0 * one)))
        z = self.logits[t].double().cpu().numpy()
        z = np.where(said + asked > 0, np.where(z > 0, z / rep, z * rep), z)
        M = np.abs(z) + 2 * np.abs(freq * said) + abs(pres)
        z = z - freq * said - pres * (said > 0)
        if self.bias is not None:
            a, e = self.bias[0][b:b + 2]
            add = np.zeros(V)
            for token, value in zip(self.bias[1][a:e], self.bias[2][a:e]):
                if 0 <= token < V:
                    add[token] = value
            z, M = z + add, M + np.where(np.isfinite(add), np.abs(add), 0)
        if self.allowed is not None:
            row = t if self.rows is None else self.rows[t]
            if row >= 0:
                bits = (self.allowed[row][:, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(-1)[:V]
                z = np.where(bits > 0, z, -np.inf)
        return z, 5 * E32 * M + 2.0 ** -149

    def check(self, out, chosen):
        _, u, least = TYPES[self.dtype]
        got = out.double().cpu().numpy()
        for t in range(self.starts[-1]):
            z, tol = self.reference(t)
            fine = np.isfinite(z)
            assert (got[t][~fine] == -np.inf).all()
            assert (np.abs(got[t] - z)[fine] <= (tol + u * (np.abs(z) + tol) + least)[fine]).all(), t
            if chosen is None:
                continue
            c = int(chosen[t])
            if not fine.any():
                assert c == -1
                continue
            assert 0 <= c < self.V and fine[c]
            best = int(np.argmax(np.where(fine, z, -np.inf)))
            assert z[c] + tol[c] >= z[best] - tol[best], (t, c, best)
            if c != best:  # a tie as far as fp32 can tell
                assert z[best] - z[c] <= tol[c] + tol[best] and (z[c] < z[best] or c < best)
        rest = slice(int(self.starts[-1]), None)
        assert (got[rest] == 7).all() and (chosen is None or (chosen[rest] == 77).all())


CASES = [
    dict(counts=[1], V=1, dtype="fp32"),
    dict(counts=[1], V=1000, dtype="fp32", biases=5),
    dict(counts=[1], V=262144, dtype="fp32", history=(500, 500), biases=5),
    dict(counts=[16, 3, 9], V=4096, dtype="fp32", trees=True, grammar="some", biases=30),
    dict(counts=[2, 0, 1, 33], V=4097, dtype="fp16", trees=True, grammar="some", biases=300, padding=3),
    dict(counts=[1] * 40, V=5003, dtype="bf16", grammar="some", history=(0, 3000)),
    dict(counts=[5, 1, 4], V=100003, dtype="bf16", trees=True, grammar="own", history=(0, 30000), biases=40),
    dict(counts=[3, 2], V=8191, dtype="fp16", history=(0, 0), biases=2000, padding=1),
    dict(counts=[64, 2], V=2049, dtype="fp32", trees=True, history=(0, 1)),
    dict(counts=[256], V=300, dtype="bf16", trees=True, grammar="some", history=(900, 900)),
    dict(counts=[7, 7], V=33, dtype="fp32", grammar="nothing", biases=9),
    dict(counts=[9], V=70001, dtype="fp16", factors=False, trees=True),
    dict(counts=[4, 4], V=31, dtype="bf16", prompt=1.0),
    dict(counts=[4, 4], V=12289, dtype="fp32", prompt=0.0, trees=True),
    # the largest vocabulary, and more different tokens than are counted at once
    dict(counts=[2, 1], V=393216, dtype="fp16", history=(60000, 60000), biases=3000, grammar="some"),
    dict(counts=[1, 3], V=393213, dtype="fp32", history=(50000, 60000), biases=3000, trees=True),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_logit_rules(cuda, case):
    rows = Rows(seed=case, **CASES[case])
    rows.check(*rows.run())
    no_device_error()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("V,offset,pad", [(4096, 0, 0), (4096, 1, 0), (5000, 3, 1), (4099, 0, 5), (97, 2, 3)])
def test_rows_of_any_alignment_in_place_and_by_another_stream(cuda, dtype, V, offset, pad):
    """Rows that begin anywhere and lie apart; out being logits; the same bits however it is called."""
    rows = Rows([3, 1, 2], V, dtype, history=(0, 200), biases=20, grammar="some", trees=True, seed=V + offset)
    ref, chosen = rows.run()
    rows.check(ref, chosen)
    T = len(rows.logits)
    wide = torch.full((T, V + offset + pad + 9), 5.0, dtype=rows.logits.dtype, device="cuda")
    view = wide[:, offset:offset + V]
    view.copy_(rows.logits)
    out = torch.full((T, V + offset + pad), 5.0, dtype=rows.logits.dtype, device="cuda")
    for o in (out[:, pad:pad + V], torch.empty_like(rows.logits)):
        got, again = rows.run(out=o, logits=view, stream=torch.cuda.Stream())
        assert torch.equal(got, ref) and torch.equal(again, chosen)
    got, again = rows.run(out=view, logits=view)
    assert torch.equal(got, ref) and torch.equal(again, chosen)
    assert (wide[:, :offset] == 5).all() and (wide[:, offset + V:] == 5).all()
    assert (out[:, :pad] == 5).all() and (out[:, pad + V:] == 5).all()
    got, none = rows.run(tokens=False)
    assert torch.equal(got, ref) and none is None
    no_device_error()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ties_infinities_and_nan(cuda, dtype):
    """Equal logits go to the lowest token, across chunks and lanes; infinities stay what they are; NaN is
    never chosen; a row of NaN and -infinity has no token."""
    V = 20000
    rows = Rows([10], V, dtype, history=(0, 0), factors=False)
    z = rows.logits
    z.zero_()
    z[1, 17000] = z[1, 17001] = z[1, 4100] = 9.0
    z[2, 3] = float("inf")
    z[2, 4] = float("nan")
    z[3] = float("-inf")
    z[4] = float("nan")
    z[5] = -torch.arange(V, device="cuda") - 1.0
    z[6] = float("-inf")
    z[6, V - 1] = torch.finfo(z.dtype).min
    z[7, 5], z[7, 0] = -0.0, -1.0
    z[8, :18000], z[9, :18000] = -1.0, -1.0
    z[8, 17], z[9, 18003] = -0.0, -0.0
    out, chosen = rows.run()
    assert torch.equal(out.nan_to_num(3.0), z.nan_to_num(3.0)) and torch.equal(out.isnan(), z.isnan())
    # (-0 is below +0 in no comparison: the lower token of the two)
    assert chosen.tolist() == [0, 4100, 3, -1, -1, 0, V - 1, 1, 17, 18000]


def test_the_quotient_is_that_of_fp32(cuda):
    """Any bits of a logit and of a repetition penalty: the same as the fp32 division and product by themselves,
    bit for bit (NaN: some NaN; a zero keeps no sign, since a bias of 0 is added)."""
    V, rng = 50000, np.random.default_rng(11)
    reps = np.concatenate([rng.integers(0, 2 ** 32, 20, dtype=np.uint64).astype(np.uint32).view(np.float32),
                           np.float32([1.1, 1.3, 3, 1e-38, 1e-45, 3e38, 0, -2, np.inf, np.nextafter(np.float32(1), 2)])])
    B = len(reps)
    rows = Rows([1] * B, V, "fp32", history=(V, V), prompt=1.0, factors=False)
    rows.history[:] = np.arange(V)
    rows.rep = reps
    z = rng.integers(0, 2 ** 32, (B, V), dtype=np.uint64).astype(np.uint32).view(np.float32)
    z[:, :V // 2] = (rng.standard_normal((B, V // 2)) * 10).astype(np.float32)
    rows.logits.copy_(torch.from_numpy(z))
    out, _ = rows.run()
    with np.errstate(all="ignore"):
        want = np.where(z > 0, z / reps[:, None], z * reps[:, None])
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    no_device_error()


def test_quotients_half_way_between_the_smallest_numbers(cuda):
    """Odd multiples of half the penalty, in steps of 2^-149: every quotient lies on a middle and goes to the
    even neighbour."""
    V, reps = 4000, np.float32([98, 150, 196, 206, 334, 6, 1022, 3998])
    rows = Rows([1] * len(reps), V, "fp32", history=(V, V), prompt=1.0, factors=False)
    rows.history[:] = np.arange(V)
    rows.rep = reps
    odd = np.arange(1, 2 * V, 2)
    z = (odd[None] * (reps[:, None].astype(np.int64) // 2) * 2.0 ** -149).astype(np.float32)
    rows.logits.copy_(torch.from_numpy(z))
    out, _ = rows.run()
    np.testing.assert_array_equal(out.cpu().numpy(), z / reps[:, None])
    no_device_error()


def test_the_last_bias_of_a_token_counts(cuda):
    rows = Rows([1, 1], 100, "fp32", history=(0, 0), factors=False)
    rows.bias = (np.array([0, 4, 7]), np.array([5, 5, 9, 5, 9, 100, -1]), np.array([1, 2, 3, 40, 50, 6, 7], np.float32))
    out, chosen = rows.run()
    rows.check(out, chosen)
    assert chosen.tolist() == [5, 9] and torch.equal(out[0, 5], rows.logits[0, 5] + 40)


def test_rules_in_a_graph(cuda):
    """Captured once, replayed with other logits, histories and masks in the same places."""
    from edgeexpert_b200.sampling import LogitRules
    op, rows = LogitRules(), Rows([2, 3], 9000, "fp32", history=(100, 100), trees=True, seed=4)
    starts, history, lens, prompt = i32(rows.starts), i32(rows.history), i32(rows.lens), i32(rows.prompt)
    rep, pres, freq = (torch.from_numpy(x).cuda() for x in (rows.rep, rows.pres, rows.freq))
    ids, bits = i32(rows.drafted), words_of(rows.masks, 1)
    out, tokens = torch.zeros_like(rows.logits), i32(np.zeros(5))
    ws = torch.empty(op.workspace_bytes(5, 9000, 2, 100), dtype=torch.uint8, device="cuda")

    def call():
        op.encode(rows.logits, out, starts, ws, max_query=3, history=history, history_lens=lens, prompt_lens=prompt,
                  repetition=rep, presence=pres, frequency=freq, token_ids=ids, ancestors=bits, tokens=tokens)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        now = Rows([2, 3], 9000, "fp32", history=(0, 100), trees=True, seed=10 + seed)
        for to, x in ((rows.logits, now.logits), (history, i32(now.history)), (lens, i32(now.lens)),
                      (prompt, i32(now.prompt)), (rep, torch.from_numpy(now.rep)), (pres, torch.from_numpy(now.pres)),
                      (freq, torch.from_numpy(now.freq)), (ids, i32(now.drafted)), (bits, words_of(now.masks, 1))):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        now.check(out, tokens)


def test_calls_at_once_and_no_rows(cuda):
    """Two batches on two streams at the same time, each with a workspace of its own; a batch of no rows."""
    from edgeexpert_b200.sampling import LogitRules
    op, calls = LogitRules(), []
    for rows in (Rows([3, 30, 1], 50001, "bf16", history=(0, 3000), seed=1), Rows([1] * 9, 70000, "fp32", history=(9, 90), seed=2)):
        want, chosen = rows.run()
        ws = torch.empty(rows.workspace(op, len(rows.logits)), dtype=torch.uint8, device="cuda")
        kw = dict(history=i32(rows.history), history_lens=i32(rows.lens), prompt_lens=i32(rows.prompt), max_query=30)
        kw.update((n, torch.from_numpy(x).cuda()) for n, x in (("repetition", rows.rep), ("presence", rows.pres),
                                                               ("frequency", rows.freq)))
        outs = [(torch.full_like(rows.logits, 7.0), i32(np.full(len(rows.logits), 77))) for _ in range(20)]
        calls.append((rows, want, chosen, ws, kw, i32(rows.starts), torch.cuda.Stream(), outs))
    torch.cuda.synchronize()
    for i in range(20):
        for rows, _, _, ws, kw, starts, stream, outs in calls:
            op.encode(rows.logits, outs[i][0], starts, ws, tokens=outs[i][1], stream=stream, **kw)
    torch.cuda.synchronize()
    for _, want, chosen, *_, outs in calls:
        assert all(torch.equal(o, want) and torch.equal(t, chosen) for o, t in outs)
    z = torch.zeros(0, 64, device="cuda")
    op.encode(z, z, i32([0, 0]), calls[0][3], tokens=i32([]))
    no_device_error()


def test_lists_that_the_kernel_bounds(cuda):
    """Rows beyond the bound, masks that do not exist, lengths beyond their lists: reported or cut, not read."""
    rows = Rows([4, 2], 500, "fp32", history=(5, 5), biases=3)
    ref, chosen = rows.run()
    out, some = rows.run(max_query=2)
    assert flags() and torch.equal(out[[0, 1, 4, 5]], ref[[0, 1, 4, 5]]) and (out[2:4] == 7).all()
    assert torch.equal(some[[0, 1, 4, 5]], chosen[[0, 1, 4, 5]]) and (some[2:4] == 77).all()
    rows.lens = np.array([10 ** 6, -3])
    out, _ = rows.run()
    rows.lens = np.array([5, 0])
    rows.check(out, None)
    rows.bias = (np.array([-5, rows.bias[0][1], 10 ** 6]),) + rows.bias[1:]
    out, _ = rows.run()
    rows.bias = (np.array([0, rows.bias[0][1], len(rows.bias[1])]),) + rows.bias[1:]
    rows.check(out, None)
    no_device_error()
    rows = Rows([2, 2], 500, "fp32", grammar="some")
    rows.rows = np.array([0, 1, 2, -9])  # (two masks)
    out, chosen = rows.run()
    assert flags()
    rows.rows = np.array([0, 1, -1, -1])
    rows.check(out, chosen)
    no_device_error()


def test_refusals(cuda):
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.sampling import LogitRules
    op = LogitRules()
    z = torch.zeros(4, 64, device="cuda")
    ws = torch.empty(op.workspace_bytes(4, 64, 2, 4, 1), dtype=torch.uint8, device="cuda")
    two = i32([1, 1])

    def call(logits=z, out=None, starts=i32([0, 2, 4]), ws=ws, max_query=2, tokens=i32([0] * 4), **kw):
        op.encode(logits, torch.empty_like(logits) if out is None else out, starts, ws, max_query=max_query,
                  tokens=tokens, **kw)

    call()
    f = torch.ones(2, device="cuda")
    bits = i32(np.zeros((4, 1)))
    for bad in (dict(logits=z.double()), dict(out=z.half()), dict(out=z[:, :63]), dict(logits=z.t(), out=z.t()),
                dict(logits=z[0]), dict(starts=torch.tensor([0, 2, 4], device="cuda")), dict(starts=i32([0])),
                dict(max_query=0), dict(ws=ws[:8]), dict(tokens=i32([0] * 3)), dict(tokens=torch.zeros(4).cuda()),
                dict(history=i32([[1], [2]])), dict(history_lens=two), dict(prompt_lens=two),
                dict(history=i32([[1]]), history_lens=two), dict(history=torch.zeros(2, 1).cuda(), history_lens=two),
                dict(history=i32(np.zeros((2, 4))).t()[:2], history_lens=two), dict(repetition=torch.ones(3, device="cuda")),
                dict(repetition=f.double()), dict(presence=f.cpu()), dict(bias_starts=i32([0, 1, 1])),
                dict(bias_starts=i32([0, 1, 1]), bias_tokens=i32([1]), bias_values=f),
                dict(bias_starts=i32([0, 1]), bias_tokens=i32([1]), bias_values=f[:1]),
                dict(allowed=i32(np.zeros((4, 1)))), dict(allowed=i32(np.zeros((3, 2)))), dict(allowed_rows=i32([0] * 4)),
                dict(allowed=i32(np.zeros((4, 2))), allowed_rows=i32([0] * 3)), dict(token_ids=i32([0] * 4)),
                dict(ancestors=bits), dict(token_ids=i32([0] * 4), ancestors=bits[:3]),
                dict(token_ids=i32([0] * 4), ancestors=bits[:, :0]), dict(token_ids=i32([0] * 4), ancestors=bits.cpu()),
                dict(logits=z.cpu(), out=z.cpu())):
        with pytest.raises(TFError):
            call(**bad)
    call(history=i32([[1], [2]]), history_lens=two, repetition=f, allowed=i32(np.zeros((4, 2))))
    no_device_error()
