"""Tables, chunk attention and windows together, as a server uses them: requests that arrive,
run prompts in chunks beside others' decoding, roll drafts back and finish, through quantized
projections and several layers, against one KvCache a request."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from unillm_amd import F16, KvCache, PagedKvCache, PageTable, QuantLinear  # noqa: E402

pytestmark = pytest.mark.gpu

H, KVH, HD, LAYERS, HIDDEN = 8, 2, 64, 2, 192
WIDTH = (H + 2 * KVH) * HD


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def linear(n, k, g):
    w = (torch.randn(n, k, generator=g) * k ** -0.5).half()
    return QuantLinear.from_blocks(F16, n, k, w.numpy().view(np.uint8).reshape(-1))


@pytest.fixture(scope="module")
def layers():
    g = torch.Generator().manual_seed(0)
    return [(linear(WIDTH, HIDDEN, g), linear(HIDDEN, H * HD, g)) for _ in range(LAYERS)]


def forward(layers, x, attend):
    for i, (qkv, o) in enumerate(layers):
        x = x + o.forward(attend(i, qkv.forward(x)))
    return x


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 4e-3), (torch.float16, 1.4e-2), (torch.bfloat16, 1.1e-1)])
def test_requests_come_run_and_go(layers, dtype, tol):
    # Tolerances, with q, k, v of order 1.  f32: KvCache forms its angles in f32, each up to
    # 112 * 2^-23 off, on q and on k; the pairs' frequencies fall by 0.75 a pair, so 4 pairs' worth
    # of |q||k| / sqrt(hd) <= 2 each: a score is off by 2e-4, an output by 2 * 4 (|v|) times that,
    # and two layers of projections of unit gain: 4e-3.  16 bits: each key's element is half a step
    # off at most, a score by 64 independent roundings, 0.6 half steps over sqrt(hd) of their root
    # sum: 0.6 half steps, and an output by as much in each layer; twelve deviations, in two layers
    # (each the sum of k's and v's): 12 * 0.6 * 2 * 2 half steps of 2^-11 or 2^-8 = 1.4e-2, 1.1e-1.
    g = torch.Generator().manual_seed(3)
    r = np.random.RandomState(1)
    page = 16
    table = PageTable(4, 20, 40, page, 128)
    paged = [PagedKvCache(KVH, HD, 40, page, dtype) for _ in range(LAYERS)]
    slots, waiting = [None] * 4, [int(n) for n in (70, 3, 41, 100, 16, 7, 33, 58)]
    finished = 0
    step = 0
    while finished < 8:
        step += 1
        assert step < 200
        for i in range(4):  # requests arrive
            if slots[i] is None and waiting:
                slots[i] = {"prompt": waiting.pop(0), "done": 0, "caches": [KvCache(KVH, HD, 320) for _ in range(LAYERS)]}
        batch = [i for i in r.permutation(4) if slots[i] is not None and (r.rand() < 0.9 or step % 7 == 0)]
        if not batch:
            continue
        news = []
        for i in batch:  # a chunk of the prompt, or a token, or drafted tokens
            left = slots[i]["prompt"] - slots[i]["done"]
            news.append(min(left, int(r.randint(1, 40))) if left > 0 else int(r.choice([1, 1, 4])))
        x = [torch.randn(n, HIDDEN, generator=g).cuda() for n in news]
        table.extend(ints(batch), ints(news))
        got = forward(layers, torch.cat(x), lambda l, qkv: paged[l].attention(table, qkv, H))
        first = 0
        for i, n, xi in zip(batch, news, x):
            want = forward(layers, xi, lambda l, qkv: slots[i]["caches"][l].attention(qkv, H))
            assert (got[first:first + n] - want).abs().max().item() <= tol, (step, i)
            first += n
            slots[i]["done"] += n
        # drafts rolled back
        back = [(i, int(r.randint(1, n))) for i, n in zip(batch, news) if n == 4 and r.rand() < 0.7]
        if back:
            keep = [slots[i]["done"] - b for i, b in back]
            table.truncate(ints([i for i, _ in back]), ints(keep))
            for (i, _), k in zip(back, keep):
                slots[i]["done"] = k
                for c in slots[i]["caches"]:
                    c.truncate(k)
        gone = [i for i in range(4) if slots[i] is not None and slots[i]["done"] >= slots[i]["prompt"] + 12]
        if gone:
            table.release(ints(gone))
            for i in gone:
                slots[i] = None
            finished += len(gone)
        table.check()
        held = sum(-(-s["done"] // page) for s in slots if s is not None)
        assert table.n_free.item() == 40 - held
    assert table.n_free.item() == 40 - sum(-(-s["done"] // page) for s in slots if s is not None)


def test_a_window_equals_the_whole_while_it_covers_the_sequence(layers):
    g = torch.Generator().manual_seed(5)
    table = PageTable(2, 10, 20, 16, 100)
    caches = [PagedKvCache(KVH, HD, 20, 16, torch.float16) for _ in range(LAYERS)]
    for n in ([80, 20], [1, 1], [9, 0]):
        table.extend(ints([1, 0]), ints(n))
        x = torch.randn(sum(n), HIDDEN, generator=g).cuda()
        a = forward(layers, x, lambda l, qkv: caches[l].attention(table, qkv, H))
        b = forward(layers, x, lambda l, qkv: caches[l].attention(table, qkv, H, window=90, sinks=4))
        assert torch.equal(a, b)
    table.check()
