"""GPU tests of PagedDecoder where requests are refused, lists are short and
batches are small, against the contiguous decoder on each sequence by itself.

Two layers, each within 2e-3 of the formulas on either side: 8e-3 between
them, as for the whole path in test_gpu_paged.py."""
import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_paged import f64, i32, no_device_error

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    """(weights, last hidden states of a sequence by position)."""
    from edgeexpert_b200.decoder import Decoder, DecoderConfig, KVCache, synthetic_decoder
    cfg = DecoderConfig(d=256, f=128, fs=128, num_experts=16, top_k=8, num_q_heads=4, num_kv_heads=2, head_dim=64,
                        vocab=1000, layers=2, max_context=64)
    dev = torch.device("cuda", 0)
    weights = synthetic_decoder(cfg, dev, torch.Generator(device=dev).manual_seed(7))

    def alone(tokens):
        dec = Decoder(weights, 1, KVCache(cfg, 1, dev))
        rows = []
        for pos, token in enumerate(tokens):
            dec.step(i32([token]), pos)
            rows.append(f64(dec.h)[0].copy())
        return rows

    return weights, alone


def paged(weights, requests, pages, max_pages, T, page_size, max_query):
    from edgeexpert_b200.paged import PagedDecoder, PagedKVCache
    cfg = weights.cfg
    cache = PagedKVCache(cfg.layers, cfg.num_kv_heads, cfg.head_dim, requests, pages, max_pages, T, page_size=page_size)
    return PagedDecoder(weights, T, cache, max_query=max_query), cache


def close(row, want):
    assert O.rel_error(row.astype(np.float32), want.astype(np.float32)) < 8e-3


def padded(tokens, T):
    ids = np.zeros(T, np.int64)
    ids[:len(tokens)] = tokens
    return i32(ids)


class Users:
    """Users whose tokens are offered until they are granted."""

    def __init__(self, model, sizes, T, **kw):
        rng = np.random.default_rng(sum(sizes))
        self.weights, alone = model
        self.tokens = [rng.integers(1, 1000, n) for n in sizes]
        self.want = [alone(t) for t in self.tokens]
        self.at, self.T = [0] * len(sizes), T
        self.dec, self.cache = paged(self.weights, len(sizes), T=T, **kw)

    def offer(self, targets, granted):
        """A step to `targets`, of which exactly the requests in `granted` come about; the list
        holds the tokens of every request that grows, as far as it goes."""
        ids = np.concatenate([t[o:max(o, n)] for t, o, n in zip(self.tokens, self.at, targets)] + [np.zeros(0, np.int64)])
        self.dec.step(padded(ids[:self.T], self.T), i32(targets))
        grown = [(b, j) for b in granted for j in range(self.at[b], targets[b])]
        asked = sum(n > o for o, n in zip(self.at, targets))
        assert self.cache.free_state.tolist()[2:] == [asked - len(granted), len(grown)]
        for b, n in enumerate(targets):
            if b in granted or 0 <= n < self.at[b]:
                self.at[b] = n
        assert self.cache.seq_lens.tolist() == self.at
        h = f64(self.dec.h)
        for row, (b, j) in enumerate(grown):
            close(h[row], self.want[b][j])
        no_device_error()


def test_a_refused_request_leaves_the_others_their_tokens(cuda, model):
    """No page for a request in the middle and for the last one: those granted behind the first
    get their own tokens, and the refused ones later."""
    u = Users(model, [6, 6, 6, 3], T=12, pages=4, max_pages=3, page_size=4, max_query=4)
    u.offer([4, 4, 3, 0], [0, 1, 2])
    u.offer([5, 5, 4, 2], [0, 2])    # one free page: the first takes it, the third needs none
    u.offer([6, 5, 5, 2], [0])
    u.offer([0, 5, 5, 2], [])        # the first is finished; its pages can be taken from the next step on
    u.offer([-1, 5, 5, 2], [1, 2])
    u.offer([-1, 6, 6, -1], [1, 2])


def test_a_request_longer_than_its_table_is_refused_alone(cuda, model):
    u = Users(model, [3, 13, 4], T=16, pages=16, max_pages=3, page_size=4, max_query=13)
    u.offer([2, 13, 1], [0, 2])      # 13 positions are more than three pages hold; its tokens are in the list
    u.offer([3, 12, 1], [0, 1])


def test_tokens_that_the_list_does_not_hold_are_not_added(cuda, model):
    """The list ends at T tokens: a request whose tokens lie behind is refused, also where the
    tokens before it are refused too and its own would fit."""
    u = Users(model, [12, 6, 4], T=12, pages=2, max_pages=2, page_size=8, max_query=12)
    u.offer([0, 1, 0], [1])
    u.offer([10, 6, 2], [])          # no two pages for the first; the second's five are at 10..14 of the list
    u.offer([7, 6, 2], [0, 1])       # the third's are at 12 and 13


def test_lists_of_any_length_up_to_the_step(cuda, model):
    """A list shorter than the step is the whole list: nothing behind it is read."""
    u = Users(model, [9, 5], T=12, pages=16, max_pages=3, page_size=4, max_query=9)
    whole = torch.full((40,), 10 ** 6, dtype=torch.int32, device="cuda")  # no token of the vocabulary behind the list
    for targets in ([4, 1], [5, 2], [-1, 3], [-1, -1], [9, 5], [0, 0]):
        ids = np.concatenate([t[o:max(o, n)] for t, o, n in zip(u.tokens, u.at, targets)])
        whole[:len(ids)] = i32(ids)
        u.dec.step(whole[:len(ids)], i32(targets))
        rows = [(b, j) for b in range(2) for j in range(u.at[b], targets[b])]
        h = f64(u.dec.h)
        for row, (b, j) in enumerate(rows):
            close(h[row], u.want[b][j])
        u.at = [o if n < 0 else n for o, n in zip(u.at, targets)]
        assert u.cache.seq_lens.tolist() == u.at
    # any negative target leaves a request alone
    u.dec.step(i32(u.tokens[0][:3]), i32([3, -1]))
    u.dec.step(i32(u.tokens[1][:2]), torch.tensor([-2 ** 31, 2], dtype=torch.int32, device="cuda"))
    assert u.cache.seq_lens.tolist() == [3, 2] and u.cache.free_state.tolist()[2:] == [0, 2]
    u.dec.step(i32([]), i32([0, 0]))
    # a request whose tokens the short list does not hold is refused
    u.dec.step(i32(u.tokens[0][:3]), i32([2, 2]))
    assert u.cache.seq_lens.tolist() == [2, 0] and u.cache.free_state.tolist()[2:] == [1, 2]
    no_device_error()


def test_step_refusals(cuda, model):
    from edgeexpert_b200._lib import TFError
    dec, cache = paged(model[0], 2, T=12, pages=8, max_pages=3, page_size=4, max_query=4)
    for ids, targets in ((torch.zeros(12, dtype=torch.int64, device="cuda"), i32([1, 1])), (i32(np.zeros(13)), i32([1, 1])),
                         (i32(np.zeros((3, 4))), i32([1, 1])), (torch.zeros(12, dtype=torch.int32), i32([1, 1])),
                         (i32(np.zeros(12)), i32([1])), (i32(np.zeros(12)), torch.tensor([1, 1], device="cuda")),
                         (i32(np.zeros(12)), torch.ones(2, dtype=torch.int32))):
        with pytest.raises(TFError):
            dec.step(ids, targets)
    assert cache.seq_lens.tolist() == [0, 0] and cache.free_state.tolist()[1] == 8
    no_device_error()


def test_steps_that_the_lm_head_cannot_take(cuda, model):
    """Refused before anything is written, not at the end of the first step."""
    from edgeexpert_b200._lib import TFError
    for T in (0, 257):
        with pytest.raises(TFError):
            paged(model[0], 2, T=T, pages=80, max_pages=70, page_size=4, max_query=T)
    dec, cache = paged(model[0], 1, T=256, pages=64, max_pages=64, page_size=4, max_query=256)
    dec.step(i32(np.arange(256)), i32([256]))
    assert cache.seq_lens.tolist() == [256] and ((dec.tokens >= 0) & (dec.tokens < 1000)).all()
    no_device_error()


def test_a_prefix_shared_on_a_raw_stream(cuda, model):
    """An integer names a stream here as it does in every other call."""
    u = Users(model, [9, 12], T=12, pages=16, max_pages=3, page_size=4, max_query=12)
    u.dec.step(i32(u.tokens[0][:6]), i32([6, -1]))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    u.cache.share(0, 6, stream=stream.cuda_stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert u.cache.prefix_len == 6 and u.cache.seq_lens.tolist() == [0, 0]
    u.dec.step(i32(u.tokens[0][6:]), i32([3, -1]))
    for row in range(3):
        close(f64(u.dec.h)[row], u.want[0][6 + row])
    no_device_error()


class Watched:
    """A decoder whose routing inputs and choices are kept, layer by layer."""

    def __init__(self, dec):
        self.dec, self.layers, moe = dec, [], dec._moe

        def watched(i, stream):
            moe(i, stream)
            self.layers.append((dec.router_x.cpu().numpy().copy(), dec.idx.cpu().numpy().copy()))

        dec._moe = watched

    def step(self, *args):
        self.layers.clear()
        self.dec.step(*args)
        return f64(self.dec.h), list(self.layers)


def bits(t):
    t = t.contiguous()
    return t.view(torch.int16).cpu().numpy().view(np.uint16) if t.is_floating_point() else t.cpu().numpy()


@pytest.mark.parametrize("T", [1, 2, 5, 8])
def test_steps_of_a_few_tokens(cuda, model, T):
    """Up to eight rows the projections are GEMVs, and one row has its own path through the experts.

    The choice of experts is not continuous: two states within the tolerance of each other may
    choose differently where two logits nearly meet.  There the choice is checked against the
    formula on the row's own state in 64 bits, and the row's result has nothing to be compared with."""
    from edgeexpert_b200.decoder import Decoder, KVCache
    weights, cfg, dev = model[0], model[0].cfg, torch.device("cuda", 0)
    rng = np.random.default_rng(16)
    users = [rng.integers(1, 1000, n) for n in (7, 9)]
    want = []
    for user in users:
        dec = Watched(Decoder(weights, 1, KVCache(cfg, 1, dev)))
        want.append([dec.step(i32([token]), pos) for pos, token in enumerate(user)])
    dec, cache = paged(weights, 2, T=T, pages=16, max_pages=3, page_size=4, max_query=T)
    dec, at, apart, compared = Watched(dec), [0, 0], set(), 0
    while at != [7, 9]:
        added, targets = [], []
        for b in range(2):
            n = min(T - len(added), len(users[b]) - at[b])
            targets.append(at[b] + n if n else -1)
            added += [(b, j) for j in range(at[b], at[b] + n)]
            at[b] += n
        h, layers = dec.step(i32([users[b][j] for b, j in added]), i32(targets))
        for row, (b, j) in enumerate(added):
            (ho,), theirs = want[b][j]
            for i, ((x, idx), (xo, idxo)) in enumerate(zip(layers, theirs)):
                if b in apart:
                    break
                close(f64(torch.from_numpy(x[row])), f64(torch.from_numpy(xo[0])))
                if set(idx[row]) != set(idxo[0]):
                    M = weights.layers[i].moe
                    logits = O.router_logits(bits(M.router_w), bits(M.router_s), bits(M.router_b),
                                             x[row].view(np.uint16), bits(M.eff_scale))[1]
                    chosen = np.isin(np.arange(cfg.num_experts), idx[row])
                    # (fp32 sums of 256 products)
                    assert logits[chosen].min() >= logits[~chosen].max() - 256 * 2.0 ** -23 * np.abs(logits).max()
                    if i + 1 < cfg.layers:  # what later tokens of the request see of it is different too
                        apart.add(b)
                    break
            else:
                if b not in apart:
                    close(h[row], ho)
                    compared += 1
    assert compared >= 12  # of sixteen
    no_device_error()
