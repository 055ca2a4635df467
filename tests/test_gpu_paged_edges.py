"""GPU tests of the serving operators at the edges of what their callers may
pass: what rows do not see, bounds that are not met, views, tokens outside
every request.  References and tolerances are those of test_gpu_paged.py."""
import ctypes as C

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


# a window that ends behind the prefix for every row, for some, and one that ends inside it
OUT_OF_SIGHT = [([70, 61, 90], [1, 2, 4], 16, 4, 128, "bf16", 50), ([60] * 40, [1] * 40, 16, 8, 256, "fp16", 60),
                ([80, 200, 66], [1, 66, 1], 16, 8, 64, "fp16", 14), ([30], [1], 2, 2, 320, "fp16", 20),
                ([3, 9, 40], [1, 1, 1], 16, 8, 256, "fp16", 40)]


@pytest.mark.parametrize("case", range(len(OUT_OF_SIGHT)))
def test_prefix_pages_that_no_row_sees(cuda, case):
    """Page ids of the prefix that lie out of every row's window may be anything (the pages have
    been given to others): nothing is reported and nothing is read."""
    lens, counts, nq, nkv, hd, dtype, window = OUT_OF_SIGHT[case]
    batch = Batch(700, lens, counts, nq, nkv, hd, dtype, 16, seed=40 + case)
    first = min(max(0, 700 + n - c - window + 1) for n, c in zip(lens, counts))  # the first position any row sees
    batch.prefix_pages = batch.prefix_pages.copy()
    batch.prefix_pages[:first // 16] = -1
    out, lse = batch.run(window)
    no_device_error()
    batch.check(out, lse, window)


def test_more_queries_than_announced_under_a_window(cuda):
    """Tokens beyond max_query give 0 and the error bit; those within it are right, wherever they stand."""
    from edgeexpert_b200._lib import Context, TFError
    batch = Batch(200, [2, 30], [40, 1], 8, 4, 64, "fp16", 16, seed=50)
    out, lse = batch.run(window=20, max_query=3)
    with pytest.raises(TFError):
        Context.get(0).check_device()
    assert (out[3:40] == 0).all() and (lse[3:40] == -float("inf")).all()
    shared, own = f64(batch.both[0]), f64(batch.both[1])
    keys, values = (np.concatenate([shared[i], own[i]]) for i in (0, 1))
    ro, rl, A, s = attention_reference(f64(batch.q[:3]), keys, values, 200 + 2 - 40 + np.arange(3), batch.scale, 20)
    u = U[torch.float16]
    assert (np.abs(f64(out[:3]) - ro) <= (2 * u + 2 * s + 16 * E32) * A + 242 * 2.0 ** -25 * 6 + 2.0 ** -25).all()
    assert (np.abs(f64(lse[:3]) - rl) <= s + 300 * E32 + 8 * E32 * np.abs(rl) + 4 * E32).all()
    no_device_error()


def test_rope_frequencies_of_a_view(cuda):
    """Frequencies are read side by side: a view with gaps is refused."""
    from edgeexpert_b200._lib import TFError
    from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
    z = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros(2, 4, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    gaps = torch.ones(64, dtype=torch.float64, device="cuda")[::2]
    with pytest.raises(TFError):
        RotaryKVWrite().encode(z, z, z, torch.empty_like(z), PagedKV(kc, vc), i32([0, 1]), i32([0, 1]), gaps)


@pytest.mark.parametrize("switch", ["0", "1", None])
def test_dependent_launches_can_be_switched_off(cuda, monkeypatch, switch):
    """TFCUDA_PDL=0 holds for these operators as for all others: no edge between two of their
    kernels is a programmatic one."""
    from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
    batch = Batch(100, [20, 30], [1, 1], 8, 4, 64, "fp16", 16, seed=70)
    op, kv = SharedPrefixAttention(), PagedKV(batch.k, batch.v)
    ws = torch.empty(op.workspace_bytes(kv, 8, 2, 2, 100, 1), dtype=torch.uint8, device="cuda")
    args = (i32(batch.table), i32(batch.lens), i32(batch.starts))
    pages, out, lse = i32(batch.prefix_pages), torch.zeros_like(batch.q), torch.zeros(2, 8, device="cuda")

    def call():
        op.encode(batch.q, kv, *args, out, ws, prefix_pages=pages, prefix_len=100, lse=lse)

    monkeypatch.delenv("TFCUDA_PDL", raising=False)
    if switch is not None:
        monkeypatch.setenv("TFCUDA_PDL", switch)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
        call()
    raw, count = C.c_void_p(int(graph.raw_cuda_graph())), C.c_size_t(0)
    edges = C.CDLL("libcuda.so.1").cuGraphGetEdges_v2
    assert edges(raw, None, None, None, C.byref(count)) == 0 and count.value == 3  # four kernels in a row
    ends, data = [(C.c_void_p * 3)() for _ in range(2)], (C.c_uint8 * 24)()  # data: 8 bytes an edge, the third its type
    assert edges(raw, *ends, data, C.byref(count)) == 0
    assert [data[8 * i + 2] for i in range(3)] == [0 if switch == "0" else 1] * 3
    out.zero_()
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    batch.check(out, lse)
