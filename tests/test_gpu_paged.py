"""GPU tests of the serving operators (page tables of a ragged batch, rotary
positions with the paged cache write, attention behind a shared prefix)
against plain implementations in 64 bits.

Tolerances, with u the unit roundoff of the 16-bit type (2^-11 fp16, 2^-8
bf16) and e = 2^-24 that of fp32:
* whole numbers are equal;
* rotation: one rounding u|y| of the result, plus at most 16 fp32 roundings of
  terms no larger than the pair's |a| + |b| (the norm, its weight, the angle's
  cosine and sine, products and sum), plus half of fp16's smallest step;
* attention, with A = sum p|v| / sum p: weights may be rounded to 16 bits (u A),
  the result is (u A at most), and every score may be off by s = (dim + 16) e
  max(sum |q k|) scale, which moves both sums by a factor e^s (2 s A); weights
  below fp16's normal range lose up to 2^-25 each (keys * 2^-25 max|v|).
  lse: s, plus a rounding for each addition of the sum, plus its own."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def i32(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).cuda()


def f64(t):
    return t.double().cpu().numpy()


def no_device_error():
    from edgeexpert_b200._lib import Context
    assert Context.get(torch.cuda.current_device()).check_device() == 0


# ------------------------------------------------------------------ pages ----
class Sequential:
    """The page tables' rules, one request after another."""

    def __init__(self, lens, table, ring, head, count, ps):
        self.lens, self.table, self.ring, self.head, self.count, self.ps = list(lens), table, ring, head, count, ps

    def resize(self, targets, max_tokens, base):
        ps, N, width = self.ps, len(self.ring), self.table.shape[1]

        def pages(n):
            return -(-n // ps)

        asked = asked_tokens = taken = back = refused = 0
        starts, slots, positions, requests = [0], [], [], []
        lens, head, count = list(self.lens), self.head, self.count
        given = []
        for b, t in enumerate(targets):
            o = lens[b]
            if 0 <= t < o:
                given += [self.table[b, j] for j in range(pages(t), pages(o))]
                self.lens[b] = t
            elif t > o:
                ok = t <= width * ps
                if ok:
                    need = pages(t) - pages(o)
                    asked += need
                    ok = need == 0 or asked <= count
                    if ok:
                        asked_tokens += t - o
                        ok = asked_tokens <= max_tokens
                if ok:
                    for j in range(need):
                        self.table[b, pages(o) + j] = self.ring[(head + asked - need + j) % N]
                    taken = asked if need else taken
                    self.lens[b] = t
                    for s in range(o, t):
                        slots.append(self.table[b, s // ps] * ps + s % ps)
                        positions.append(base + s)
                        requests.append(b)
                else:
                    refused += 1
            starts.append(len(slots))
        for j, page in enumerate(given):
            self.ring[(head + count + j) % N] = page
        self.head, self.count = (head + taken) % N, count - taken + len(given)
        pad = [-1] * (max_tokens - len(slots))
        return starts, slots + pad, positions + pad, requests + pad, [self.head, self.count, refused, len(slots)]


def random_pool(rng, B, ps, width, lens, spare):
    held = [-(-n // ps) for n in lens]
    N = max(1, sum(held) + spare)
    ids = rng.permutation(N)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    head = int(rng.integers(N))
    ring = np.full(N, -1, np.int32)
    for j, page in enumerate(ids[at:]):
        ring[(head + j) % N] = page
    return table, ring, head, N - at


class PagesOnGpu:
    def __init__(self, seq, max_tokens):
        from edgeexpert_b200.paged import KVPages
        B = len(seq.lens)
        self.op, self.max_tokens, self.ps = KVPages(), max_tokens, seq.ps
        self.lens, self.table, self.ring = i32(seq.lens), i32(seq.table), i32(seq.ring)
        self.state = i32([seq.head, seq.count, 0, 0])
        self.starts = i32(np.full(B + 1, -7))
        self.slots, self.positions, self.requests = (i32(np.full(max_tokens, -7)) for _ in range(3))
        self.ws = torch.empty(KVPages.workspace_bytes(B), dtype=torch.uint8, device="cuda")

    def resize(self, targets, base, lens_out=None, state_out=None, stream=None):
        self.op.encode_resize(self.lens, targets, self.table, self.ring, self.state,
                              self.lens if lens_out is None else lens_out,
                              self.state if state_out is None else state_out, self.starts, self.slots, self.positions,
                              self.requests, self.ps, self.ws, position_base=base, stream=stream)


def assert_pages(gpu, seq, answer, lens=None, state=None):
    starts, slots, positions, requests, want = answer
    assert gpu.starts.tolist() == starts
    assert gpu.slots.tolist() == slots
    assert gpu.positions.tolist() == positions
    assert gpu.requests.tolist() == requests
    assert (gpu.lens if lens is None else lens).tolist() == seq.lens
    assert (gpu.state if state is None else state).tolist() == want
    assert np.array_equal(gpu.table.cpu().numpy(), seq.table)
    assert np.array_equal(gpu.ring.cpu().numpy(), seq.ring)


def make_targets(rng, lens, grow, width, ps):
    targets = []
    for o in lens:
        kind = rng.random()
        if kind < 0.1:
            targets.append(0)
        elif kind < 0.2:
            targets.append(-1 if rng.random() < 0.5 else o)
        elif kind < 0.3:
            targets.append(int(rng.integers(0, o + 1)))
        elif kind < 0.33:
            targets.append(width * ps + int(rng.integers(1, 5)))
        else:
            targets.append(o + int(rng.integers(1, grow + 1)))
    return targets


@pytest.mark.parametrize("B,ps,old,grow,spare,max_tokens", [
    (1, 16, 0, 1, 4, 1), (1, 1, 5, 300, 400, 300), (2, 16, 40, 1, 8, 7), (31, 17, 100, 4, 20, 200),
    (32, 16, 64, 1, 0, 32),          # no free page: only requests with room in their last page grow
    (33, 128, 1000, 500, 30, 9000),  # pages run out on the way
    (100, 8, 60, 40, 2000, 700),     # tokens run out on the way
    (1000, 16, 50, 3, 300, 3000), (2500, 4, 9, 9, 2000, 20000), (64, 16, 30, 2000, 9000, 0)])
def test_pages_resize(cuda, B, ps, old, grow, spare, max_tokens):
    rng = np.random.default_rng(B * 1000 + ps)
    lens = [int(rng.integers(0, old + 1)) for _ in range(B)]
    width = -(-(old + grow) // ps)
    seq = Sequential(lens, *random_pool(rng, B, ps, width, lens, spare), ps)
    gpu = PagesOnGpu(seq, max_tokens)
    targets = make_targets(rng, lens, grow, width, ps)
    # with separate outputs the call can be repeated
    lens_out, state_out = i32(np.zeros(B)), i32(np.zeros(4))
    for _ in range(2):
        gpu.resize(i32(targets), 1000, lens_out, state_out)
    assert_pages(gpu, seq, seq.resize(targets, max_tokens, 1000), lens_out, state_out)
    no_device_error()


@pytest.mark.parametrize("B,ps", [(5, 16), (40, 3)])
def test_pages_over_many_steps_in_place(cuda, B, ps):
    """A serving loop on another stream, in place: requests come, grow, are cut
    back and finish; no page is ever lost or held twice."""
    rng = np.random.default_rng(B)
    width = 12
    seq = Sequential([0] * B, *random_pool(rng, B, ps, width, [0] * B, B * width // 2), ps)
    N = len(seq.ring)
    gpu = PagesOnGpu(seq, 5 * B)
    stream = torch.cuda.Stream()
    for step in range(30):
        targets = make_targets(rng, seq.lens, 6, width, ps)
        t = i32(targets)
        torch.cuda.synchronize()
        gpu.resize(t, 0, stream=stream)
        stream.synchronize()
        assert_pages(gpu, seq, seq.resize(targets, 5 * B, 0))
        held = [p for b in range(B) for p in seq.table[b, :-(-seq.lens[b] // ps)]]
        free = [seq.ring[(seq.head + j) % N] for j in range(seq.count)]
        assert sorted(held + free) == list(range(N))
    no_device_error()


def test_pages_resize_refusals(cuda):
    from edgeexpert_b200._lib import TFError
    rng = np.random.default_rng(0)
    seq = Sequential([3, 4], *random_pool(rng, 2, 4, 3, [3, 4], 2), 4)

    def call(**change):
        g = PagesOnGpu(seq, 8)
        a = dict(lens=g.lens, targets=i32([4, 5]), table=g.table, ring=g.ring, state=g.state, lens_out=g.lens,
                 state_out=g.state, starts=g.starts, slots=g.slots, positions=g.positions, requests=g.requests,
                 page=4, ws=g.ws, base=0)
        a.update(change)
        g.op.encode_resize(a["lens"], a["targets"], a["table"], a["ring"], a["state"], a["lens_out"], a["state_out"],
                           a["starts"], a["slots"], a["positions"], a["requests"], a["page"], a["ws"], a["base"])

    call()
    for bad in (dict(targets=i32([4])), dict(lens=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(page=0),
                dict(ws=torch.empty(8, dtype=torch.uint8, device="cuda")), dict(starts=i32([0, 0])),
                dict(table=i32([[1, 2, 3]])), dict(state=i32([0, 1])), dict(positions=i32([0])),
                dict(page=0x7FFFFFFF), dict(base=0x7FFFFFFF)):
        with pytest.raises(TFError):
            call(**bad)


# ------------------------------------------------------------------- rope ----
def rope_reference(q, k, v, positions, freq, factor, layout, q_weight, k_weight, norm, eps):
    """-> (q, k, v) in 64 bits and, per value, the size its fp32 roundings scale with."""
    half = len(freq)
    angle = positions[:, None].astype(np.float64) * freq[None]
    cos, sin = np.cos(angle)[:, None] * factor, np.sin(angle)[:, None] * factor

    def normed(x, w):
        if norm:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
            x = x if w is None else x * w
        return x

    def turned(x):
        y, size = x.copy(), np.abs(x)
        a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
        size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * factor
        return y, size

    v = normed(v, None)
    return turned(normed(q, q_weight)), turned(normed(k, k_weight)), (v, np.abs(v))


ROPE = [
    # T, nq, nkv, hd, rot, layout, norm, dtype, page, longest position
    (1, 16, 8, 256, 256, "half", True, "fp16", 16, 4096),
    (1, 16, 8, 256, 256, "interleaved", False, "bf16", 1, 2 ** 31 - 1),
    (7, 16, 2, 64, 64, "half", True, "bf16", 17, 131072),
    (33, 8, 1, 128, 64, "interleaved", True, "fp16", 64, 1 << 20),
    (5, 4, 4, 512, 128, "half", True, "fp16", 8, 4096),
    (3, 12, 4, 80, 36, "half", True, "fp16", 16, 999),       # pairs that no vector boundary meets
    (3, 12, 4, 80, 50, "interleaved", False, "bf16", 16, 999),
    (130, 1, 1, 8, 8, "half", False, "fp16", 16, 50),
    (65, 0, 2, 64, 64, "half", True, "bf16", 16, 4096),      # K and V alone
    (19, 6, 2, 24, 0, "half", True, "fp16", 4, 100),         # norms and cache write without rotation
    (300, 16, 8, 256, 128, "half", False, "fp16", 16, 4096),
]


@pytest.mark.parametrize("T,nq,nkv,hd,rot,layout,norm,dtype,page,longest", ROPE)
@pytest.mark.parametrize("form", ["apart", "fused", "by head"])
def test_rope_kv_write(cuda, T, nq, nkv, hd, rot, layout, norm, dtype, page, longest, form):
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
    dt, rng = DT[dtype], np.random.default_rng(T + hd + rot)
    gen = torch.Generator(device="cuda").manual_seed(T * hd)

    def normal(*shape):
        return (torch.randn(*shape, device="cuda", generator=gen) * 3).to(dt)

    if form == "fused":
        qkv = normal(T, (nq + 2 * nkv) * hd)
        q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    else:
        q, k, v = normal(T, nq, hd), normal(T, nkv, hd), normal(T, nkv, hd)
    pages = -(-T // page) + 3
    if form == "by head":  # K and V of a page together, heads outside positions
        pool = torch.full((pages, 2, nkv, page, hd), 7.0, dtype=dt, device="cuda")
        kc, vc = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    else:
        kc, vc = (torch.full((pages, page, nkv, hd), 7.0, dtype=dt, device="cuda") for _ in range(2))
    slots = rng.permutation(pages * page)[:T]
    positions = rng.integers(0, longest, T)
    positions[0] = longest
    padding = rng.random(T) < 0.2 if T > 1 else np.zeros(T, bool)
    slots[padding], positions[padding] = -1, -1
    freq = 10000.0 ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))
    factor = 1.0 if layout == "half" else 1.25
    weights = [(1 + 0.2 * torch.randn(hd, device="cuda", generator=gen)).to(torch.bfloat16) if norm else None
               for _ in range(2)]
    refs = rope_reference(f64(q), f64(k), f64(v), positions, freq, factor, layout,
                          *[None if w is None else f64(w) for w in weights], norm, 1e-6)
    q_out = q if form == "fused" else torch.full_like(q, 7.0)  # in place too
    RotaryKVWrite().encode(q, k, v, q_out, PagedKV(kc, vc), i32(slots), i32(positions),
                           torch.tensor(freq, device="cuda"), rotary_dim=rot, layout=layout, attention_factor=factor,
                           q_weight=weights[0], k_weight=weights[1], norm=norm)
    torch.cuda.synchronize()

    def close(got, ref, size):
        assert (np.abs(got - ref) <= U[dt] * np.abs(ref) + 16 * E32 * size + 2.0 ** -25).all()

    live = ~padding
    got = f64(q_out)
    if nq:
        close(got[live], refs[0][0][live], refs[0][1][live])
        assert (got[padding] == 0).all()
    for cache, (ref, size) in ((kc, refs[1]), (vc, refs[2])):
        flat = f64(cache).reshape(pages * page, nkv, hd)
        close(flat[slots[live]], ref[live], size[live])
        untouched = np.ones(pages * page, bool)
        untouched[slots[live]] = False
        assert (flat[untouched] == 7.0).all()
    no_device_error()


def test_rope_unaligned_rows(cuda):
    """Rows that start at odd elements: token strides and bases of 2-byte alignment."""
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
    T, nq, nkv, hd = 9, 4, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(5)
    buf = torch.randn(T, (nq + 2 * nkv) * hd + 3, device="cuda", generator=gen).half()
    q, k, v = (x.unflatten(1, (-1, hd))
               for x in buf[:, 1:-2].split([nq * hd, nkv * hd, nkv * hd], 1))
    kc, vc = (torch.zeros(2, 8, nkv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    pos, freq = np.arange(T) * 100, 10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)
    q_out = torch.zeros(T, nq * hd + 1, dtype=torch.float16, device="cuda")[:, 1:].unflatten(1, (nq, hd))
    RotaryKVWrite().encode(q, k, v, q_out, PagedKV(kc, vc), i32(np.arange(T)), i32(pos), torch.tensor(freq, device="cuda"))
    ref = rope_reference(f64(q), f64(k), f64(v), pos, freq, 1.0, "half", None, None, False, 0.0)
    for got, (want, size) in ((q_out, ref[0]), (kc.flatten(0, 1)[:T], ref[1]), (vc.flatten(0, 1)[:T], ref[2])):
        assert (np.abs(f64(got) - want) <= U[torch.float16] * np.abs(want) + 16 * E32 * size + 2.0 ** -25).all()


def test_rope_agrees_with_the_contiguous_epilogue(cuda):
    """At one position with every pair turned it is tf_qkv_epilogue, which rounds
    the norm to fp16 first: one more half ulp of each of the pair's values."""
    from edgeexpert_b200.decoder import FusedQKVEpilogue
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite, rope_frequencies
    T, nq, nkv, hd, position = 3, 16, 8, 256, 1234
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(T, n, hd, device="cuda", generator=gen).half() for n in (nq, nkv, nkv))
    qw, kw = ((1 + 0.1 * torch.randn(hd, device="cuda", generator=gen)).to(torch.bfloat16) for _ in range(2))
    kc, vc = (torch.zeros(1, T, nkv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    q_out = torch.empty_like(q)
    freq, factor = rope_frequencies(hd)
    RotaryKVWrite().encode(q, k, v, q_out, PagedKV(kc, vc), i32(range(T)), i32([position] * T), freq,
                           attention_factor=factor, q_weight=qw, k_weight=kw, norm=True)
    FusedQKVEpilogue().encode(q, k, v, qw, kw, hd, nq, nkv, T, position, 10000.0, hd // 2)
    for got, want in ((q_out, q), (kc[0], k), (vc[0], v)):
        # fp32 angles there: position * 2^-24 radians of the pair on top
        g, w = f64(got), f64(want)
        size = np.abs(w) + np.abs(np.roll(w, hd // 2, -1))
        assert (np.abs(g - w) <= (4 * 2.0 ** -11 + 4 * position * E32) * size + 2.0 ** -24).all()


def test_rope_refusals(cuda):
    from edgeexpert_b200._lib import Context, TFError
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
    T, hd = 2, 64
    z = torch.zeros(T, 4, hd, dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros(2, 4, 4, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    kv, freq = PagedKV(kc, vc), torch.ones(hd // 2, dtype=torch.float64, device="cuda")

    def call(q=z, k=z, q_out=None, slots=i32([0, 1]), freq=freq, **kw):
        RotaryKVWrite().encode(q, k, z, torch.empty_like(z) if q_out is None else q_out, kv, slots, i32([0, 1]), freq, **kw)

    call()
    for bad in (dict(q=z.bfloat16()), dict(slots=i32([0])), dict(freq=freq.float()), dict(freq=freq[:8]),
                dict(layout="spiral"), dict(k=z[:, :2]), dict(q=z.transpose(1, 2)), dict(rotary_dim=63),
                dict(rotary_dim=128, freq=torch.ones(64, dtype=torch.float64, device="cuda")),
                dict(norm=True, eps=-1.0), dict(q_weight=torch.ones(hd, device="cuda"))):
        with pytest.raises(TFError):
            call(**bad)
    # a slot beyond the pool is reported and skipped
    call(k=z + 1, slots=i32([8, 1]))
    with pytest.raises(TFError):
        Context.get(0).check_device()
    turned = torch.cat([torch.full((hd // 2,), np.cos(1.0) - np.sin(1.0)), torch.full((hd // 2,), np.cos(1.0) + np.sin(1.0))])
    assert (kc[0, 0] == 0).all() and torch.equal(kc[0, 1], turned.half().cuda().expand(4, hd))
    no_device_error()


# -------------------------------------------------------------- attention ----
def attention_reference(q, keys, values, at, scale, window):
    """One request: q [n][nq][hd], keys / values [positions][nkv][hd] (prefix and
    own), at[n] the positions of the queries.  -> out, lse, A, the score bound."""
    n, nq, hd = q.shape
    P, nkv, _ = keys.shape
    out, lse, A = np.zeros((n, nq, hd)), np.full((n, nq), -np.inf), np.zeros((n, nq, hd))
    most = 0.0
    for j in range(n):
        lo = max(0, at[j] - window + 1) if window else 0
        hi = min(P, at[j] + 1)
        if hi <= lo:
            continue
        for h in range(nq):
            k, v = keys[lo:hi, h * nkv // nq], values[lo:hi, h * nkv // nq]
            s = (k @ q[j, h]) * scale
            most = max(most, float((np.abs(k) @ np.abs(q[j, h])).max()) * scale)
            w = np.exp(s - s.max())
            out[j, h], A[j, h] = (w @ v) / w.sum(), (w @ np.abs(v)) / w.sum()
            lse[j, h] = s.max() + np.log(w.sum())
    return out, lse, A, (hd + 16) * E32 * most


class Batch:
    """A ragged batch in a pool whose unused places hold NaN."""

    def __init__(self, prefix, lens, counts, nq, nkv, hd, dtype, page, seed=0, by_head=False, padding=0, q_std=1.5):
        self.dt, self.P, self.page = DT[dtype], prefix, page
        gen = torch.Generator(device="cuda").manual_seed(seed * 1000 + prefix + hd)
        rng = np.random.default_rng(seed)
        self.lens, self.counts = list(lens), list(counts)
        B, T = len(lens), sum(counts) + padding
        held = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        total = shared + sum(held) + 2
        ids = rng.permutation(total)

        def pool():
            shape = (total, nkv, page, hd) if by_head else (total, page, nkv, hd)
            t = torch.full(shape, float("nan"), dtype=self.dt, device="cuda")
            return t.transpose(1, 2) if by_head else t

        self.k, self.v = pool(), pool()
        self.keys, self.values = [], []
        self.prefix_pages = ids[:shared]
        width = max(1, max(held))
        self.table = np.full((B, width), -1)
        at = shared
        both = [torch.randn(2, prefix, nkv, hd, device="cuda", generator=gen).to(self.dt)]
        self._store(both[0], self.prefix_pages)
        for b in range(B):
            self.table[b, :held[b]] = ids[at:at + held[b]]
            own = torch.randn(2, lens[b], nkv, hd, device="cuda", generator=gen).to(self.dt)
            self._store(own, ids[at:at + held[b]])
            both.append(own)
            at += held[b]
        self.both = both
        self.q = (torch.randn(T, nq, hd, device="cuda", generator=gen) * q_std).to(self.dt)
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        self.scale = hd ** -0.5

    def _store(self, kv, pages):
        for i in range(0, kv.shape[1], self.page):
            n = min(self.page, kv.shape[1] - i)
            self.k[pages[i // self.page], :n] = kv[0, i:i + n]
            self.v[pages[i // self.page], :n] = kv[1, i:i + n]

    def run(self, window=0, max_query=None, stream=None, out=None, lse=True, q=None):
        from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
        op, kv = SharedPrefixAttention(), PagedKV(self.k, self.v)
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
            op.encode(q, kv, *args, out, ws, prefix_pages=prefix, prefix_len=self.P, max_query=mq, scale=self.scale,
                      window=window, lse=lse, stream=stream)
            torch.cuda.synchronize()
            answers.append(out.clone())
        assert torch.equal(answers[0].view(torch.int16), answers[1].view(torch.int16))
        return out, lse

    def check(self, out, lse, window=0):
        out, lse, q, u = f64(out), f64(lse), f64(self.q), U[self.dt]
        shared = f64(self.both[0])
        for b, (length, n) in enumerate(zip(self.lens, self.counts)):
            own = f64(self.both[1 + b])
            keys, values = (np.concatenate([shared[i], own[i]]) for i in (0, 1))
            t = slice(self.starts[b], self.starts[b + 1])
            at = self.P + length - n + np.arange(n)
            ro, rl, A, s = attention_reference(q[t], keys, values, at, self.scale, window)
            seen, N = np.isfinite(rl), len(keys)
            small = N * 2.0 ** -25 * (np.abs(values).max() if N else 0) if self.dt == torch.float16 else 0
            tol = (2 * u + 2 * s + 16 * E32) * A + small + 2.0 ** -25
            assert (np.abs(out[t] - ro) <= tol).all(), (b, np.abs(out[t] - ro).max())
            assert (lse[t][~seen] == -np.inf).all() and (out[t][~seen] == 0).all()
            err = np.abs(lse[t][seen] - rl[seen])
            assert (err <= s + N * E32 + 4 * E32 * np.abs(rl[seen]) + 4 * E32).all(), (b, err.max())
        assert (out[self.starts[-1]:] == 0).all() and (lse[self.starts[-1]:] == -np.inf).all()


ATTENTION = [
    # prefix, lens, queries, nq, nkv, hd, dtype, page, window
    (0, [1], [1], 16, 8, 256, "fp16", 16, 0),
    (1, [1, 2], [1, 1], 16, 8, 256, "fp16", 16, 0),
    (317, [1, 40], [1, 1], 16, 8, 256, "fp16", 16, 0),
    (500, [33, 1, 700, 16, 17, 128, 129], [1] * 7, 16, 8, 256, "fp16", 16, 0),
    (1023, [5, 64, 300], [1, 1, 1], 16, 4, 128, "bf16", 32, 0),
    (130, [9, 0, 31, 8], [1, 0, 4, 8], 16, 2, 64, "bf16", 17, 0),       # a request without a turn, drafts
    (64, [3, 1, 2], [5, 1, 2], 8, 1, 128, "fp16", 1, 0),                 # more queries than positions: into the prefix
    (0, [2, 0, 70], [4, 3, 2], 8, 2, 64, "fp16", 16, 0),                 # rows that see nothing
    (400, [50, 200, 3], [3, 1, 2], 12, 4, 256, "bf16", 24, 100),         # a window, over both parts
    (1500, [700, 2, 90], [1, 2, 5], 16, 8, 64, "fp16", 64, 33),          # the prefix mostly out of sight
    (300, [20, 5], [2, 1], 4, 4, 80, "fp16", 16, 0),                     # odd head sizes
    (77, [12], [1], 3, 1, 24, "bf16", 8, 0),
    (129, [40, 3], [1, 2], 4, 4, 512, "fp16", 16, 0),
    (260, [17, 30], [1, 3], 40, 1, 64, "bf16", 16, 0),                   # 40 heads to one KV head
    (200, [150, 90, 37], [150, 80, 1], 16, 8, 256, "fp16", 16, 0),       # prompts and a decode row together
    (513, [260, 131], [260, 131], 16, 4, 128, "bf16", 128, 0),
    (333, [300], [257], 8, 1, 64, "fp16", 48, 90),
    (2049, [30] * 40, [1] * 40, 16, 8, 256, "fp16", 16, 0),              # a batch that fills tensor tiles
    (900, [10 + 3 * i for i in range(70)], [1 + i % 3 for i in range(70)], 16, 2, 128, "bf16", 16, 0),
]


@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_shared_prefix_attention(cuda, case):
    prefix, lens, counts, nq, nkv, hd, dtype, page, window = ATTENTION[case]
    batch = Batch(prefix, lens, counts, nq, nkv, hd, dtype, page, seed=case, by_head=case % 3 == 1, padding=case % 4)
    out, lse = batch.run(window)
    batch.check(out, lse, window)
    no_device_error()


@pytest.mark.parametrize("counts,dtype,hd", [([1] * 24, "fp16", 256), ([40, 3, 1], "bf16", 128)])
def test_attention_of_extreme_scores(cuda, counts, dtype, hd):
    """One key far above the rest, growing scores along the keys, scores of
    hundreds below: nothing overflows and nothing is lost."""
    lens = [c + 20 for c in counts]
    batch = Batch(300, lens, counts, 16, 4, hd, dtype, 16, seed=3, q_std=20.0)
    batch.check(*batch.run())


@pytest.mark.parametrize("counts,window,hd", [([3, 1], 0, 256), ([3, 2], 40, 64), ([90, 4], 0, 128), ([1] * 40, 64, 128)])
def test_attention_of_keys_that_others_see(cuda, counts, window, hd):
    """Infinities and NaN in keys and values that only some rows of a tile see
    (the next token of a draft, a prefix position out of one row's window): the
    others are as if they were not there, and those that see them are not finite."""
    lens = [c + 13 + 5 * i for i, c in enumerate(counts)]
    batch = Batch(100, lens, counts, 8, 4, hd, "fp16", 16, seed=11)
    last = lens[0] - 1  # the last token of the first request, and a position late in the prefix
    spots = [(int(batch.table[0, last // 16]), last % 16)]
    if window:
        spots.append((int(batch.prefix_pages[75 // 16]), 75 % 16))
    for i, (page, at) in enumerate(spots):
        batch.v[page, at, :, 0] = float("inf")
        batch.v[page, at, 0, 1] = float("nan")
        batch.k[page, at, 1, 0] = float("nan")
    out, lse = (f64(x) for x in batch.run(window))
    shared = f64(batch.both[0])
    for b, (length, n) in enumerate(zip(lens, counts)):
        own = f64(batch.both[1 + b])
        keys, values = (np.concatenate([shared[i], own[i]]) for i in (0, 1))
        at = 100 + length - n + np.arange(n)
        t = slice(batch.starts[b], batch.starts[b + 1])
        ro, rl, A, s = attention_reference(f64(batch.q[t]), keys, values, at, batch.scale, window)
        hit = (at >= 100 + last) & (b == 0)
        if window:
            hit |= (at >= 75) & (at < 75 + window)
        assert (np.abs(out[t] - ro)[~hit] <= ((2 * U[torch.float16] + 2 * s + 16 * E32) * A + 1e-4)[~hit]).all()
        assert not np.isfinite(out[t][hit][..., 0]).any() and not np.isfinite(lse[t][hit][:, 2:4]).any()


def test_attention_by_another_stream_strides_and_repeats(cuda):
    """q and out as slices of wider rows, another stream, no lse; the same bits every time."""
    batch = Batch(700, [90, 5, 300], [2, 1, 3], 16, 4, 128, "fp16", 16, seed=8)
    ref, _ = batch.run()
    wide = torch.zeros(6, 24 * 128, dtype=torch.float16, device="cuda")
    wide[:, 256:256 + 2048] = batch.q.flatten(1)
    out = torch.zeros(6, 20 * 128, dtype=torch.float16, device="cuda")
    for _ in range(3):
        got, _ = batch.run(stream=torch.cuda.Stream(), lse=False, q=wide[:, 256:256 + 2048].unflatten(1, (16, 128)),
                           out=out[:, 512:512 + 2048].unflatten(1, (16, 128)))
        assert torch.equal(got, ref)
    assert (out[:, :512] == 0).all() and (out[:, 512 + 2048:] == 0).all()


def test_attention_in_a_graph(cuda):
    """Captured once, replayed with other lengths: nothing about them is fixed by the host."""
    from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
    batch = Batch(200, [100, 100], [1, 1], 16, 8, 256, "fp16", 16, seed=4)
    op, kv = SharedPrefixAttention(), PagedKV(batch.k, batch.v)
    ws = torch.empty(op.workspace_bytes(kv, 16, 2, 2, 200, 1), dtype=torch.uint8, device="cuda")
    table, lens, starts, pages = i32(batch.table), i32([100, 100]), i32(batch.starts), i32(batch.prefix_pages)
    out, lse = torch.zeros_like(batch.q), torch.zeros(2, 16, device="cuda")

    def call():
        op.encode(batch.q, kv, table, lens, starts, out, ws, prefix_pages=pages, prefix_len=200, lse=lse)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for now in ([100, 100], [1, 77], [30, 2]):
        lens.copy_(i32(now))
        graph.replay()
        torch.cuda.synchronize()
        batch.lens = now
        keep, batch.both = batch.both, [batch.both[0]] + [x[:, :n] for x, n in zip(batch.both[1:], now)]
        batch.check(out, lse)
        batch.both = keep


def test_attention_with_a_loose_bound_on_the_queries(cuda):
    """max_query far above any request's tokens changes nothing but the kernel chosen."""
    batch = Batch(150, [90, 40, 7], [70, 1, 3], 16, 4, 128, "bf16", 16, seed=21)
    for bound in (70, 1000, 2 ** 31 - 1, 2 ** 32 - 1):
        batch.check(*batch.run(max_query=bound))
    no_device_error()


def test_attention_far_into_a_pool(cuda):
    """Element offsets beyond 2^32 and byte offsets beyond 2^33."""
    from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
    nkv, hd, page = 2, 64, 16
    stride = 1 << 28
    buf = torch.empty((20 * stride) + page * nkv * hd, dtype=torch.float16, device="cuda")
    k = buf.as_strided((21, page, nkv, hd), (stride, nkv * hd, hd, 1))
    v = buf[page * nkv * hd:].as_strided((20, page, nkv, hd), (stride, nkv * hd, hd, 1))
    k = k[:20]
    batch = Batch(20, [30], [1], 4, nkv, hd, "fp16", page, seed=1)
    order = [19, 18, 17, 16]
    for i, old in enumerate(list(batch.prefix_pages) + list(batch.table[0])):
        k[order[i]], v[order[i]] = batch.k[old], batch.v[old]
    out, lse = torch.zeros_like(batch.q), torch.zeros(1, 4, device="cuda")
    op, kv = SharedPrefixAttention(), PagedKV(k, v)
    ws = torch.empty(op.workspace_bytes(kv, 4, 1, 1, 20, 1), dtype=torch.uint8, device="cuda")
    op.encode(batch.q, kv, i32([order[2:]]), i32([30]), i32([0, 1]), out, ws, prefix_pages=i32(order[:2]),
              prefix_len=20, lse=lse)
    batch.check(out, lse)


def test_attention_refusals(cuda):
    from edgeexpert_b200._lib import Context, TFError
    from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
    batch = Batch(40, [20, 30], [1, 1], 8, 4, 64, "fp16", 16)
    op, kv = SharedPrefixAttention(), PagedKV(batch.k, batch.v)
    out = torch.zeros_like(batch.q)
    ws = torch.empty(op.workspace_bytes(kv, 8, 2, 2, 40, 1), dtype=torch.uint8, device="cuda")

    def call(q=batch.q, table=None, lens=None, starts=None, out=out, ws=ws, **kw):
        kw = dict(dict(prefix_pages=i32(batch.prefix_pages), prefix_len=40), **kw)
        op.encode(q, kv, i32(batch.table) if table is None else table, i32([20, 30]) if lens is None else lens,
                  i32([0, 1, 2]) if starts is None else starts, out, ws, **kw)

    call()
    for bad in (dict(q=batch.q.bfloat16()), dict(q=batch.q[:, :6].contiguous(), out=out[:, :6].contiguous()),
                dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(max_query=0),
                dict(prefix_len=1000), dict(prefix_pages=None), dict(ws=ws[:0]), dict(starts=i32([0, 1])),
                dict(lens=torch.tensor([20, 30], device="cuda")), dict(table=i32(batch.table[:1])),
                dict(lse=torch.zeros(3, device="cuda")), dict(q=batch.q.transpose(1, 2), out=out.transpose(1, 2)),
                dict(window=1 << 31), dict(q=torch.zeros(2, 8 * 64 + 1, dtype=torch.float16, device="cuda")[:, 1:].unflatten(1, (8, 64)))):
        with pytest.raises(TFError):
            call(**bad)
    # pages outside the pool and more queries than announced are reported, not read
    for bad in (dict(table=i32(np.full_like(batch.table, 10 ** 6))), dict(prefix_pages=i32([-1, -1, -1])),
                dict(starts=i32([0, 2, 2]))):
        call(**bad)
        with pytest.raises(TFError):
            Context.get(0).check_device()
    no_device_error()


# ------------------------------------------------------------ the whole path ----
def test_paged_decoder_agrees_with_sequences_decoded_alone(cuda):
    """A shared system prompt prefilled once, three users' prompts prefilled
    together behind it, then tokens one at a time (one user finishing on the
    way), against the contiguous decoder on each whole sequence by itself.  Two
    layers, each within 2e-3 of the formulas on either side: 8e-3 between them."""
    import oracle as O
    from edgeexpert_b200.decoder import Decoder, DecoderConfig, KVCache, synthetic_decoder
    from edgeexpert_b200.paged import PagedDecoder, PagedKVCache
    cfg = DecoderConfig(d=256, f=128, fs=128, num_experts=16, top_k=8, num_q_heads=4, num_kv_heads=2, head_dim=64,
                        vocab=1000, layers=2, max_context=64)
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(7)
    weights = synthetic_decoder(cfg, dev, gen)
    rng = np.random.default_rng(3)
    prefix, users = rng.integers(0, 1000, 21), [rng.integers(0, 1000, n) for n in (6, 2, 9)]
    first = [3, 1, 5]  # of each user's tokens, the prompt

    alone = []  # the last hidden state after every position of prefix + user
    for user in users:
        dec = Decoder(weights, 1, KVCache(cfg, 1, dev))
        rows = []
        for pos, token in enumerate(np.concatenate([prefix, user])):
            dec.step(i32([token]), pos)
            rows.append(f64(dec.h)[0].copy())
        alone.append(rows)

    def close(row, want):
        assert O.rel_error(row.astype(np.float32), want.astype(np.float32)) < 8e-3

    cache = PagedKVCache(cfg.layers, cfg.num_kv_heads, cfg.head_dim, 3, 24, 6, 21, page_size=4)
    dec = PagedDecoder(weights, 21, cache, max_query=21)
    dec.step(i32(prefix), i32([21, -1, -1]))
    assert cache.free_state.tolist()[1:] == [24 - 6, 0, 21]
    for pos in range(21):
        close(f64(dec.h)[pos], alone[0][pos])
    cache.share(0, 21)

    def step(added, targets):
        ids = np.zeros(21, np.int64)
        ids[:sum(map(len, added))] = np.concatenate(added)
        dec.step(i32(ids), i32(targets))
        assert cache.free_state.tolist()[2:] == [0, sum(map(len, added))]
        return f64(dec.h)

    h = step([u[:n] for u, n in zip(users, first)], first)
    row = 0
    for u, n in enumerate(first):
        for j in range(n):
            close(h[row], alone[u][21 + j])
            row += 1
    at = list(first)
    for _ in range(4):
        live = [u for u in range(3) if at[u] < len(users[u])]
        targets = [at[u] + 1 if u in live else 0 for u in range(3)]
        h = step([users[u][at[u]:at[u] + 1] for u in live], targets)
        for row, u in enumerate(live):
            close(h[row], alone[u][21 + at[u]])
            at[u] += 1
    assert at == [6, 2, 9]
    no_device_error()
