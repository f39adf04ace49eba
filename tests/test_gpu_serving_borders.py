"""Operators of a served batch where sums nearly cancel, positions are far and batches are long, against plain implementations in 64 bits or more."""
from decimal import Decimal, localcontext

import numpy as np
import pytest
import torch

import serving_reference as ref
import test_gpu_serving as served

pytestmark = pytest.mark.gpu

BELOW_ONE = np.float32(1 - 2.0 ** -24)


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


# ---------------------------------------------------------------------------------------------- drafted tokens

@pytest.mark.parametrize("vocab", [4096, 9000, 50000])
def test_verify_of_a_refused_draft_that_had_nearly_all_the_weight(jn, vocab):
    """Looked-up drafts of probability 1 - 7e-8 and less, refused by the largest number below one: the token behind them is drawn from what little is left.  A number of
    0 takes the first index with any weight, though that is 4e-18 of the draft's and shares its chunk; others stand next to the border of every cumulative sum (the border's distance
    is 2^-25 of the sum at most, and 64-bit sums without the draft are good to 2^-45 of it)."""
    rng = np.random.default_rng(vocab)
    count = 60
    logits, tokens, u = np.full((2 * count, vocab), -np.inf, dtype=np.float32), np.zeros(2 * count, dtype=np.int64), np.zeros((2 * count, 2), dtype=np.float32)
    for s in range(count):
        r, zero = 2 * s, s % 3 == 0
        x = int(rng.integers(10, 4000 if zero else vocab - 100))
        chunk, end = x // 4096 * 4096, min(x // 4096 * 4096 + 4096, vocab)
        tokens[r + 1] = x
        logits[r, x] = 5.0
        # the rest, 1e-7 to 1e-6 of the draft's weight: over the tokens of its chunk and all others, or all behind its chunk where there are more
        near = [] if zero else rng.integers(chunk, end, 9)
        far = rng.integers(end if zero and end < vocab else x + 1 if zero else 0, vocab, 9)
        for at in np.unique(np.concatenate([near, far]).astype(int)):
            if at != x:
                logits[r, at] = np.float32(5.0 - 16.5 + 1.5 * rng.random())
        if zero:
            logits[r, x - 5] = 5.0 - 40.0
        logits[r + 1] = rng.standard_normal(vocab).astype(np.float32)
        u[r, 0], u[r + 1] = BELOW_ONE, rng.random(2)
        w = np.exp(logits[r].astype(np.float64) - 5.0)
        w[x] = 0
        c = np.cumsum(w)
        if not zero:  # the nearest number to a border, on either side of it
            border = c[rng.choice(np.nonzero(w)[0][:-1])] / c[-1]
            u[r, 1] = min(np.float32(border), BELOW_ONE)
            if s % 3 == 2:
                u[r, 1] = np.nextafter(u[r, 1], np.float32(0 if np.float64(u[r, 1]) > border else 1))
    starts, temps = np.arange(0, 2 * count + 1, 2), np.ones(count)
    want = ref.verify(logits, starts, tokens, None, temps, u)
    assert list(want[1]) == [0] * count and all(want[0][2 * s] == tokens[2 * s + 1] - 5 for s in range(0, count, 3))
    got = served.run_verify(jn, logits, starts, tokens, None, temps, u)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0]), np.argwhere(got[0] != want[0])


@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("vocab", [700, 30000])
def test_verify_of_more_rows_than_the_sums_kept(jn, with_q, vocab):
    """Sequences of 32 and more rows whose first refused draft stands around the 32nd and behind it, or nowhere; greedy ones among them."""
    rng = np.random.default_rng(vocab)
    counts, ends = [32, 33, 34, 40, 70, 70, 70, 33, 2, 64, 65], [None, None, 32, 31, 32, 33, 60, 0, None, 62, None]
    rows, starts = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    logits, tokens = (2 * rng.standard_normal((rows, vocab))).astype(np.float32), rng.integers(0, vocab, rows)
    temps = [0.0 if s % 4 == 3 else 0.8 for s in range(len(counts))]
    q = np.zeros((rows, vocab), dtype=np.float32)
    for s, (c, end) in enumerate(zip(counts, ends)):
        for j in range(c - 1):
            r, x = starts[s] + j, tokens[starts[s] + j + 1]
            logits[r, x] = 40.0 if j != end else -np.inf
            q[r] = 0.5 / vocab
            q[r, x] = 0.5
    u = rng.random((rows, 2)).astype(np.float32)
    want = ref.verify(logits, starts, tokens, q if with_q else None, temps, u)
    assert list(want[1]) == [c - 1 if e is None else e for c, e in zip(counts, ends)]
    got = served.run_verify(jn, logits, starts, tokens, q if with_q else None, temps, u)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


# ---------------------------------------------------------------------------------------------- rotary positions

def turned(theta, rot, divisor, positions):
    """Cosines and sines [positions, rot / 2] of position theta^(-2 i / rot) / divisor, the angle to 40 digits and reduced before it is a double."""
    with localcontext() as ctx:
        ctx.prec = 60
        tan = []  # arctangents of 1/5 and 1/239: pi = 16 and -4 of them (Machin)
        for n in (5, 239):
            term, total, k = Decimal(1) / n, Decimal(0), 1
            while abs(term) > Decimal(10) ** -58:
                total, term, k = total + term / k, -term / (n * n), k + 2
            tan.append(total)
        whole = 2 * (16 * tan[0] - 4 * tan[1])
        f = [(-(Decimal(2) * i / rot) * Decimal(theta).ln()).exp() / Decimal(divisor) for i in range(rot // 2)]
        angle = np.array([[float((p * x).remainder_near(whole)) for x in f] for p in positions])
    return np.cos(angle), np.sin(angle)


@pytest.mark.parametrize("theta,rot,factor", [(10000, 128, 1.0), (500000, 128, 1.0), (500000, 64, 3.0), (1000000, 250, 1.0)])
def test_rope_at_the_far_end_of_its_positions(jn, theta, rot, factor):
    """Pairs (1, 0), so that cosines and sines come out as they are.  Their angle x, up to pi / 4, is off by 2^-24 of itself for each of its conversion, its constant and its product,
    which x cos x <= 0.56 of it makes 1.7 x 2^-24 of a sine or cosine; the fraction of a turn by 2^-32, the series' last step by 2^-25, the steps before it by 0.2 x 2^-24, the terms left
    out by 2e-9: below 2.5 x 2^-24."""
    rope = jn.Rope(rot, theta=float(theta), interleaved=True, scaling="linear" if factor != 1.0 else None, factor=factor)
    pos = np.array([(1 << 31) - 1 - 977 * i for i in range(100)] + [-(1 << 31) + 1013 * i for i in range(100)] + [0, 1, -1, 131071, 1 << 27, -(1 << 27)], dtype=np.int64)
    c, s = turned(theta, rot, factor, [int(p) for p in pos])
    x = torch.zeros(len(pos), rot, device="cuda")
    x[:, 0::2] = 1
    p = torch.from_numpy(pos.astype(np.int32)).cuda()
    rope.apply_dev(x.data_ptr(), p.data_ptr(), len(pos), 1, rot, x.data_ptr())
    got = x.double().cpu().numpy()
    assert np.abs(got[:, 0::2] - c).max() <= 2.5 * 2.0 ** -24 and np.abs(got[:, 1::2] - s).max() <= 2.5 * 2.0 ** -24


# ---------------------------------------------------------------------------------------------- attention

LONG_BATCHES = [
    # hd, heads, kv, page, counts, lens, shared: more sequences than a wave has lanes, some of which have no rows, see only a part of what is shared or nothing else
    (64, 2, 1, 16, [1] * 65, [100 + i for i in range(65)], 4),
    (64, 4, 2, 32, [1, 2] * 64, [200 + 3 * i if i < 90 else 100 + i for i in range(128)], 5),
    (128, 4, 1, 16, [0] * 66 + [3] * 70 + [0, 1], [0] * 66 + [250 + i for i in range(70)] + [7, 200], 12),
    (64, 4, 4, 16, [1] * 200, [1 + (37 * i) % 240 for i in range(200)], 0),
    (192, 2, 2, 64, [2] * 129, [130 + i for i in range(129)], 2),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,page,counts,lens,shared", LONG_BATCHES)
def test_attention_of_long_batches(jn, half, hd, heads, kv, page, counts, lens, shared):
    served.test_attention(jn, half, hd, heads, kv, page, counts, lens, shared)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("top,rise,odd", [(top, rise, odd) for top in range(23, 29) for rise in (2, 4, 8, 16, 32, 64) for odd in (0, 1) if not odd or rise >= 2 ** (top - 23)])
def test_attention_of_scores_far_beyond_what_weights_hold(jn, half, top, rise, odd):
    """Scores of 2^top, or one step of FP32 above it, and `rise` above that (to the base 2), the lower ones first: the higher key has 2^rise of the weight of a lower one, and no finite
    input makes a NaN.  Where FP32 has no room for the rise the scores are equal."""
    rng = np.random.default_rng(top)
    hd, heads, kv, page, n = 64, 2, 1, 16, 700
    b = ref.Batch(rng, [1, 1], [n, n - 100], page)
    keys, values = np.zeros((n, hd), dtype=np.float32), rng.standard_normal((n, hd)).astype(np.float32).astype(np.float16).astype(np.float32)
    keys[:, 0], keys[:, 2] = 1024, 1
    keys[n // 2:, 1] = 1
    kind = torch.float16 if half else torch.float32
    pools = [torch.zeros(1, b.pages, kv, page, hd, device="cuda", dtype=kind) for _ in range(2)]
    for s in range(2):
        for p in range(b.lens[s]):
            for pool, rows in zip(pools, (keys, values)):
                pool[0, int(b.tables[s, p // page]), 0, p % page] = torch.from_numpy(rows[p]).to(kind)
    q = torch.zeros(2, heads, hd, device="cuda")
    q[:, :, 0], q[:, :, 1], q[:, :, 2] = 2.0 ** (top - 10), rise, odd * 2.0 ** (top - 23)
    got = served.run_attention(jn, b, q, pools, half, float(np.log(2.0))).double().cpu().numpy()
    base = np.float32(2.0 ** top + odd * 2.0 ** (top - 23))
    scores = (base + np.float32(rise) * keys[:, 1]).astype(np.float32).astype(np.float64)
    for s in range(2):
        z = scores[:b.lens[s]]
        w = np.exp2(z - z.max())
        want = (w / w.sum()) @ values[:b.lens[s]].astype(np.float64)
        # (weights to 2^-21, up to 700 terms added)
        assert np.abs(got[s] - want).max() <= (2.0 ** -20 + 64 * 2.0 ** -24) * np.abs(values).max()


@pytest.mark.parametrize("shift", [0.0, -7.0703125, 5.5625, -1000.5, 900.25])
def test_attention_of_many_keys_far_below_one(jn, shift):
    """FP16 pages, rows enough that spans are long: one key with all but 1e-5 of the weight in front of thousands that have 6e-10 of it each, which are the whole output.  Weights are held to
    2^-36 of the largest at least, and all of them off the same way at worst: 2^-36 a key; sums and scores 2^-12 of the result.  All scores
    are `shift` higher."""
    hd, heads, page, shared, n = 64, 64, 256, 64, 512
    long = shared * page
    rng = np.random.default_rng(0)
    b = ref.Batch(rng, [1] * n, [long + 1] * n, page, shared)
    low = -21.203125
    keys, values = torch.zeros(1, b.pages, 1, page, hd, device="cuda").half(), torch.zeros(1, b.pages, 1, page, hd, device="cuda").half()
    keys[..., 0], keys[..., 1], values[..., :] = low, shift, 1.0
    first = int(b.tables[0, 0])
    keys[0, first, 0, 0, 0], values[0, first, 0, 0] = 0.0, 0.0
    q = torch.zeros(n, heads, hd, device="cuda")
    q[..., :2] = 1.0
    nb, keep = served.batch_of(jn, b)
    cache = jn.PagedCache.wrap_dev(keys.data_ptr(), values.data_ptr(), 1, 1, hd, b.pages, page, 1)
    assert cache.attention_workspace(nb, heads) <= n * heads * 6 * (hd + 2) * 4  # (a few spans)
    got = served.run_attention(jn, b, q, [keys, values], True, 1.0).double()
    w = np.exp(low)
    want = long * w / (1 + long * w)
    assert (got - want).abs().max().item() <= long * 2.0 ** -36 + want * 2.0 ** -12


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,counts,shared", [(64, 8, 2, [1] * 40, 6), (128, 8, 1, [3, 1, 30, 2], 4), (256, 4, 2, [2] * 9, 5), (128, 4, 4, [1, 1, 1], 0)])
def test_attention_beside_queries_that_are_not_numbers(jn, half, hd, heads, kv, counts, shared):
    """NaN, infinities and the largest finite number in some rows' queries: every other row is what it is beside ordinary ones, to the bit."""
    rng = np.random.default_rng(hd)
    page = 32
    b = ref.Batch(rng, counts, [shared * page + 40 + 11 * i for i in range(len(counts))], page, shared)
    g = torch.Generator(device="cuda").manual_seed(5)
    pools = [torch.randn(1, b.pages, kv, page, hd, device="cuda", generator=g).to(torch.float16 if half else torch.float32) for _ in range(2)]
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    want = served.run_attention(jn, b, q, pools, half, 0.1)
    odd = sorted(set(int(t) for t in rng.integers(0, b.tokens, max(1, b.tokens // 6))))
    for value in (float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).max):
        other = q.clone()
        other[odd, :, ::3] = value
        got = served.run_attention(jn, b, other, pools, half, 0.1)
        rest = [r for r in range(b.tokens) if r not in odd]
        assert torch.equal(got[rest], want[rest])
        assert np.isfinite(value) or torch.isnan(got[odd]).all()


def test_two_batches_at_once(jn):
    """Append, attention and verification of two batches on two streams, each with its own cache and workspaces, beside one another: what each gives alone."""
    rng = np.random.default_rng(7)
    runs = []
    for hd, heads, kv, counts, lens, shared in ((128, 32, 8, [1] * 30, [700 + i for i in range(30)], 8), (64, 8, 2, [90, 3], [500, 40], 1)):
        b = ref.Batch(rng, counts, lens, 32, shared)
        pools = [torch.randn(1, b.pages, kv, 32, hd, device="cuda").half() for _ in range(2)]
        cache = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), 1, kv, hd, b.pages, 32, 1)
        nb, keep = served.batch_of(jn, b)
        rows, vocab = b.tokens, 20000
        qkv, q, y = torch.randn(rows, heads + 2 * kv, hd, device="cuda"), torch.empty(rows, heads, hd, device="cuda"), torch.empty(rows, heads, hd, device="cuda")
        ws = torch.empty(cache.attention_workspace(nb, heads) // 4 + 4, device="cuda")
        vs = torch.empty(jn.verify_workspace(rows, len(counts), vocab) // 4 + 4, device="cuda")
        logits, tokens = torch.randn(rows, vocab, device="cuda") * 3, torch.randint(0, vocab, (rows,), device="cuda", dtype=torch.int32)
        temps, numbers = torch.ones(len(counts), device="cuda"), torch.rand(rows, 2, device="cuda")
        out, accepted = torch.empty(rows, device="cuda", dtype=torch.int32), torch.empty(len(counts), device="cuda", dtype=torch.int32)
        rope, row = jn.Rope(hd), (heads + 2 * kv) * hd

        def run(stream, cache=cache, nb=nb, keep=keep, pools=pools, heads=heads, kv=kv, hd=hd, rows=rows, qkv=qkv, q=q, y=y, ws=ws, vs=vs, logits=logits, tokens=tokens, temps=temps,
                numbers=numbers, out=out, accepted=accepted, rope=rope, row=row, vocab=vocab, n=len(counts)):
            st = stream.cuda_stream
            cache.append_dev(0, nb, rope, heads, qkv.data_ptr(), q.data_ptr(), qkv.data_ptr() + 4 * heads * hd, qkv.data_ptr() + 4 * (heads + kv) * hd, row, 0, row, row, st)
            cache.attention_dev(0, nb, heads, q.data_ptr(), 0.1, y.data_ptr(), ws.data_ptr(), 4 * ws.numel(), stream_ptr=st)
            jn.verify_drafts_dev(logits.data_ptr(), rows, vocab, keep[1].data_ptr(), n, tokens.data_ptr(), temps.data_ptr(), numbers.data_ptr(), out.data_ptr(), accepted.data_ptr(),
                                 vs.data_ptr(), 4 * vs.numel(), stream_ptr=st)

        runs.append((run, (y, out, accepted)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    alone = []
    for (run, outs), stream in zip(runs, streams):
        run(stream)
        torch.cuda.synchronize()
        alone.append([o.clone() for o in outs])
    for _ in range(10):
        for o in [o for _, outs in runs for o in outs]:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for (run, _), stream in zip(runs, streams):
                run(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for (_, outs), was in zip(runs, alone) for a, o in zip(was, outs))
