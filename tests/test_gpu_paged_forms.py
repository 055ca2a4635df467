"""GPU tests of the serving operators in forms that take other branches: no
prefix, boxes of two and four keys, heads narrower than the tiles they are
loaded in, many requests, many rows, several tokens a CTA, steps in place.
References and tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from test_gpu_paged import (DT, E32, U, Batch, PagesOnGpu, Sequential, assert_pages, f64, i32, make_targets,
                            no_device_error, random_pool, rope_reference)

pytestmark = pytest.mark.gpu


def ragged(B, seed, longest, most):
    rng = np.random.default_rng(seed)
    counts = rng.integers(0, most + 1, B)
    return [int(n) for n in rng.integers(0, longest + 1, B) + counts], [int(n) for n in counts]


ATTENTION = {
    # prefix, lens, queries, nq, nkv, hd, dtype, page, window
    "prompts without a prefix, 256": (0, [200, 150, 37], [200, 150, 1], 16, 8, 256, "fp16", 16, 0),
    "prompts without a prefix, 128": (0, [260, 90, 70], [260, 85, 70], 16, 4, 128, "bf16", 32, 0),
    "prompts without a prefix, 64": (0, [300, 41], [257, 41], 8, 2, 64, "fp16", 8, 0),
    "prompts without a prefix, window": (0, [300, 150], [280, 150], 16, 8, 128, "bf16", 16, 100),
    "one prompt alone": (0, [129], [129], 8, 8, 256, "bf16", 16, 0),
    "decodes without a prefix": (0, [1, 700, 33, 128, 0, 16], [1, 1, 1, 1, 0, 1], 16, 8, 256, "fp16", 16, 0),
    "boxes of two": (150, [90, 30, 7], [1, 2, 1], 16, 8, 256, "fp16", 2, 0),
    "boxes of two, odd pages": (150, [90, 30, 7], [1, 2, 1], 8, 4, 64, "bf16", 6, 0),
    "boxes of two, tensor tiles": (333, [150, 20], [130, 2], 16, 8, 128, "fp16", 10, 0),
    "boxes of two, tensor tiles of 256": (131, [95] * 30, [3] * 30, 16, 8, 256, "bf16", 18, 70),
    "boxes of four": (150, [90, 30, 7], [1, 2, 1], 16, 8, 128, "fp16", 4, 0),
    "boxes of four, tensor tiles": (333, [150, 20], [130, 2], 16, 8, 64, "bf16", 12, 0),
    "boxes of four, tensor tiles of 256": (200, [150, 20], [130, 2], 16, 8, 256, "fp16", 20, 0),
    "192": (300, [50, 1, 9], [1, 1, 3], 8, 4, 192, "fp16", 16, 0),
    "192, tensor tiles": (300, [150] + [9] * 20, [140] + [1] * 20, 8, 4, 192, "bf16", 16, 0),
    "200": (100, [90, 11], [66, 2], 8, 4, 200, "fp16", 16, 0),
    "72": (100, [90, 11], [80, 2], 6, 2, 72, "bf16", 16, 0),
    "320": (200, [50, 3], [1, 2], 4, 2, 320, "fp16", 16, 0),
    "384": (90, [70, 20], [40, 3], 4, 4, 384, "bf16", 8, 30),
    "512, more rows than a job": (129, [40, 30], [23, 9], 8, 4, 512, "fp16", 16, 0),
    "600 requests": (90, *ragged(600, 1, 20, 2), 4, 2, 64, "fp16", 16, 0),
    "300 requests under a window": (70, *ragged(300, 2, 90, 3), 8, 4, 128, "bf16", 16, 40),
    "600 requests, some with prompts": (40, [70 if b % 97 == 5 else 3 for b in range(600)],
                                        [66 if b % 97 == 5 else 1 for b in range(600)], 4, 4, 64, "fp16", 8, 0),
    "16000 rows, finished and not": (90, [500, 350, 100, 9, 64], [480, 350, 100, 9, 64], 16, 8, 64, "fp16", 16, 0),
}


@pytest.mark.parametrize("name", ATTENTION)
def test_attention_forms(cuda, name):
    prefix, lens, counts, nq, nkv, hd, dtype, page, window = ATTENTION[name]
    seed = 100 + list(ATTENTION).index(name)
    batch = Batch(prefix, lens, counts, nq, nkv, hd, dtype, page, seed=seed, by_head=seed % 2 == 1, padding=seed % 3)
    out, lse = batch.run(window)
    batch.check(out, lse, window)
    no_device_error()


@pytest.mark.parametrize("T,nq,nkv,hd,rot,layout,norm,dtype,longest", [
    (2501, 8, 1, 128, 128, "half", True, "fp16", 4096), (2501, 8, 1, 128, 64, "interleaved", False, "bf16", 131072),
    (2501, 16, 2, 64, 64, "interleaved", True, "fp16", 4096), (2501, 16, 2, 64, 32, "half", True, "bf16", 999),
    (9999, 1, 1, 64, 64, "half", False, "fp16", 4096), (1301, 3, 1, 512, 512, "half", True, "fp16", 4096)])
def test_rope_of_several_tokens_a_cta(cuda, T, nq, nkv, hd, rot, layout, norm, dtype, longest):
    """In place, some rows padding, the last CTA not full."""
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
    dt, rng = DT[dtype], np.random.default_rng(T + hd + rot)
    gen = torch.Generator(device="cuda").manual_seed(T + hd)
    qkv = (torch.randn(T, (nq + 2 * nkv) * hd, device="cuda", generator=gen) * 3).to(dt)
    q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    page, pages = 24, -(-T // 24) + 3
    kc, vc = (torch.full((pages, page, nkv, hd), 7.0, dtype=dt, device="cuda") for _ in range(2))
    slots, positions = rng.permutation(pages * page)[:T], rng.integers(0, longest, T)
    padding = rng.random(T) < 0.1
    slots[padding], positions[padding] = -1, -1
    freq = 10000.0 ** (-np.arange(rot // 2) * 2.0 / rot)
    weights = [(1 + 0.2 * torch.randn(hd, device="cuda", generator=gen)).to(torch.bfloat16) if norm else None
               for _ in range(2)]
    refs = rope_reference(f64(q), f64(k), f64(v), positions, freq, 1.25, layout,
                          *[None if w is None else f64(w) for w in weights], norm, 1e-6)
    RotaryKVWrite().encode(q, k, v, q, PagedKV(kc, vc), i32(slots), i32(positions), torch.tensor(freq, device="cuda"),
                           rotary_dim=rot, layout=layout, attention_factor=1.25, q_weight=weights[0],
                           k_weight=weights[1], norm=norm)
    torch.cuda.synchronize()

    def close(got, ref, size):
        assert (np.abs(got - ref) <= U[dt] * np.abs(ref) + 16 * E32 * size + 2.0 ** -25).all()

    live, got = ~padding, f64(q)
    close(got[live], refs[0][0][live], refs[0][1][live])
    assert (got[padding] == 0).all()
    for cache, (ref, size) in ((kc, refs[1]), (vc, refs[2])):
        flat = f64(cache).reshape(pages * page, nkv, hd)
        close(flat[slots[live]], ref[live], size[live])
        untouched = np.ones(pages * page, bool)
        untouched[slots[live]] = False
        assert (flat[untouched] == 7.0).all()
    no_device_error()


@pytest.mark.parametrize("B,ps,max_tokens", [(300, 16, 900), (40, 3, 1500), (1100, 8, 4000)])
def test_pages_of_large_steps_in_place(cuda, B, ps, max_tokens):
    """The planning and the filling kernel, over steps that write the lengths and the state in place."""
    rng = np.random.default_rng(B)
    width = 12
    seq = Sequential([0] * B, *random_pool(rng, B, ps, width, [0] * B, B * width // 3), ps)
    N = len(seq.ring)
    gpu = PagesOnGpu(seq, max_tokens)
    for step in range(12):
        targets = make_targets(rng, seq.lens, 4, width, ps)
        gpu.resize(i32(targets), 5)
        assert_pages(gpu, seq, seq.resize(targets, max_tokens, 5))
        held = [p for b in range(B) for p in seq.table[b, :-(-seq.lens[b] // ps)]]
        free = [seq.ring[(seq.head + j) % N] for j in range(seq.count)]
        assert sorted(held + free) == list(range(N))
    no_device_error()
