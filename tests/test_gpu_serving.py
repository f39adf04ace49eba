"""The operators of a served batch against plain implementations in 64 bits: rotary positions, the paged cache's append and attention, the verification of
drafted tokens."""
import ctypes as C

import numpy as np
import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


def dev(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def batch_of(jn, b):
    """The package's batch and the tensors it points into."""
    keep = [dev(b.tables), dev(b.starts), dev(np.asarray(b.lens, dtype=np.int32))]
    return jn.Batch(len(b.counts), b.tokens, max([1] + b.counts), b.max_len, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr(), b.shared), keep


# ---------------------------------------------------------------------------------------------- rotary positions

ROPES = [(None, {}), ("linear", dict(factor=4.0)), ("yarn", dict(factor=8.0, original_context=4096)), ("factors", {})]


@pytest.mark.parametrize("kind,args", ROPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (80, 32), (96, 48), (6, 4), (7, 2), (256, 250)])
def test_rope(jn, kind, args, interleaved, hd, rot):
    rng = np.random.default_rng(hd + rot)
    factors = (1 + 7 * rng.random(rot // 2)).astype(np.float32) if kind == "factors" else None
    rope = jn.Rope(rot, theta=5e5, interleaved=interleaved, scaling=None if kind == "factors" else kind, freq_factors=factors, **args)
    f, m = ref.rope_frequencies(rot, 5e5, kind, args.get("factor", 1.0), args.get("original_context", 0), factors=factors)
    heads, pos = 5, np.array([0, 1, 2, 17, 4095, 131071, 1 << 20, (1 << 31) - 1, -1, -100000, -(1 << 31), 3, 3], dtype=np.int32)
    x = rng.standard_normal((len(pos), heads, hd)).astype(np.float32)
    want, bound = ref.rotate(x, pos, f, m, interleaved), ref.rotation_bound(x, f, m, interleaved)
    # (angles of positions near 2^31 are off by 2^-53 of themselves in the reference as well)
    bound = bound + (np.abs(pos.astype(np.float64)) * 2.0 ** -52)[:, None, None] * 2 * m * np.abs(x).max()
    stride, shift = heads * hd + 3, 1  # rows that are aligned to nothing
    for dense in (True, False):
        xs = dev(x) if dense else torch.zeros(len(pos) * stride + shift, device="cuda")
        if not dense:
            torch.as_strided(xs, (len(pos), heads * hd), (stride, 1), shift).copy_(dev(x).reshape(len(pos), -1))
        y = torch.full_like(xs, 7.0)
        p = dev(pos)
        rope.apply_dev(xs.data_ptr() + (0 if dense else 4 * shift), p.data_ptr(), len(pos), heads, hd, y.data_ptr() + (0 if dense else 4 * shift),
                       0 if dense else stride, 0 if dense else stride)
        got = y if dense else torch.as_strided(y, (len(pos), heads, hd), (stride, hd, 1), shift)
        assert (np.abs(got.cpu().numpy().astype(np.float64).reshape(x.shape) - want) <= bound).all()
        if not dense:  # nothing between the rows
            assert y[0] == 7 and (torch.as_strided(y, (len(pos) - 1, 3), (stride, 1), shift + heads * hd) == 7).all()
        rope.apply_dev(xs.data_ptr() + (0 if dense else 4 * shift), p.data_ptr(), len(pos), heads, hd, xs.data_ptr() + (0 if dense else 4 * shift),
                       0 if dense else stride, 0 if dense else stride)
        assert torch.equal(xs if dense else torch.as_strided(xs, (len(pos), heads, hd), (stride, hd, 1), shift), got)  # in place


def test_rope_refusals(jn):
    from jitnn_amd import _lib
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=2048), dict(rot_dim=8, theta=0.0), dict(rot_dim=8, theta=float("nan")), dict(rot_dim=8, scaling="linear", factor=0.0),
                dict(rot_dim=8, scaling="yarn", factor=2.0), dict(rot_dim=8, scaling="yarn", factor=2.0, original_context=10, beta_fast=0.5),
                dict(rot_dim=8, freq_factors=[1, 1, 0, 1]), dict(rot_dim=8, freq_factors=[1, 1]), dict(rot_dim=8, scaling="dynamic"), dict(rot_dim=8, attention_factor=-1.0)):
        with pytest.raises(ValueError):
            jn.Rope(**bad)
    r = jn.Rope(8)
    x = torch.zeros(64, device="cuda")
    call = _lib.lib.jitnn_hip_rope_dev
    p = x.data_ptr()
    assert call(None, p, 16, p, 1, 2, 8, p, 16, None) == _lib.EINVAL
    assert call(r.handle, p, 16, p, 1, 2, 6, p, 16, None) == _lib.EINVAL       # rot_dim beyond the head
    assert call(r.handle, p, 15, p, 1, 2, 8, p, 16, None) == _lib.EINVAL       # rows that overlap
    assert call(r.handle, p, 16, p, 1, 2, 8, p, 20, None) == _lib.EINVAL       # in place, another stride
    assert call(r.handle, p, 16, p, -1, 2, 8, p, 16, None) == _lib.EINVAL
    assert call(r.handle, None, 16, p, 1, 2, 8, p, 16, None) == _lib.EINVAL
    assert call(r.handle, None, 16, None, 0, 2, 8, None, 16, None) == 0        # no tokens


# ---------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,rot,interleaved,page", [(64, 8, 2, 64, True, 16), (128, 32, 8, 128, False, 64), (192, 5, 5, 96, False, 256), (256, 3, 1, 256, True, 32),
                                                              (128, 0, 4, 128, False, 16), (64, 70, 10, 0, False, 128)])
def test_append(jn, half, hd, heads, kv, rot, interleaved, page):
    """Ragged rows, sequences without any, rows behind the last sequence, a position below 0, positions outside the table and pages that do not exist."""
    rng = np.random.default_rng(hd + heads)
    b = ref.Batch(rng, [1, 0, 37, 4, 1, 2], [1, 5, 270, 3, 77, 1000], page, pad_rows=5, max_len=900)
    b.tables[4, 76 // page] = b.pages            # a page that the cache does not have
    b.tables[2, 260 // page] = -1                # and one for the rows from position 256 on
    layers, layer = 3, 1
    kind = torch.float16 if half else torch.float32
    g = torch.Generator(device="cuda").manual_seed(hd)
    pools = [torch.randn(layers, b.pages, kv, page, hd, device="cuda", generator=g).to(kind) for _ in range(2)]
    cache = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), layers, kv, hd, b.pages, page, 1 if half else 0)
    row = (heads + 2 * kv) * hd
    x = rng.standard_normal((b.tokens, heads + 2 * kv, hd)).astype(np.float32)
    x[3, heads] = 1e30                            # beyond FP16: its largest
    x[3, -1, 0] = -1e5
    x[4, -1, 1], x[4, -1, 2] = np.inf, 1e-7
    qkv = dev(x)
    rope = jn.Rope(rot, theta=1e4, interleaved=interleaved, scaling="linear", factor=2.0) if rot else None
    f, m = ref.rope_frequencies(rot, 1e4, "linear", 2.0) if rot else (np.zeros(0), 1.0)
    nb, keep = batch_of(jn, b)
    before = [p.clone() for p in pools]
    q_out = torch.full((b.tokens, max(heads, 1), hd), 7.0, device="cuda")
    base = qkv.data_ptr()
    cache.append_dev(layer, nb, rope, heads, base, q_out.data_ptr(), base + 4 * heads * hd, base + 4 * (heads + kv) * hd, q_stride=row, k_stride=row, v_stride=row)
    pos_of = np.zeros(b.tokens)
    for r, s, p in b.places():
        pos_of[r] = p
    turned, bound = ref.rotate(x[:, : heads + kv], pos_of, f, m, interleaved), ref.rotation_bound(x[:, : heads + kv], f, m, interleaved)
    want, slack = [p.double().cpu().numpy() for p in before], [np.zeros(p.shape) for p in before]
    written = set()
    for r, s, p in b.places():
        if p < 0 or p // page >= b.width or not 0 <= b.tables[s, p // page] < b.pages:
            continue
        written.add(r)
        at = (layer, b.tables[s, p // page], slice(None), p % page)
        want[0][at], want[1][at], slack[0][at] = turned[r, heads:], x[r, heads + kv:], bound[r, heads:]
    assert 20 < len(written) < b.starts[-1]
    got_q = q_out.double().cpu().numpy()
    for r in range(b.tokens):
        if heads and r in written:
            assert (np.abs(got_q[r] - turned[r, :heads]) <= bound[r, :heads]).all()
        else:
            assert (got_q[r] == 7).all()
    for i, p in enumerate(pools):
        got, w, off = p.double().cpu().numpy(), want[i], slack[i]
        if half:  # half a step of FP16 beside the rotation's own; beyond its range the largest finite value
            beyond = (np.abs(w) > 65504 + off) & np.isfinite(w)
            w = np.where(beyond, np.sign(w) * 65504, w)
            off = np.where(beyond, 0, off + np.where(np.isfinite(w), np.abs(w), 0) * 2.0 ** -11 + 2.0 ** -25)
        with np.errstate(invalid="ignore"):
            same = (got == w) | (np.abs(got - w) <= off)
        assert same.all(), np.argwhere(~same)[:4]
        rest = np.ones(got.shape, dtype=bool)
        for r, s, pp in b.places():
            if r in written:
                rest[(layer, b.tables[s, pp // page], slice(None), pp % page)] = False
        assert np.array_equal(got[rest], before[i].double().cpu().numpy()[rest])  # and nothing else was touched


def test_append_in_place_and_page_copies(jn):
    rng = np.random.default_rng(5)
    hd, heads, kv, page = 64, 4, 2, 16
    b = ref.Batch(rng, [20, 3], [20, 40], page)
    cache = jn.PagedCache(2, kv, hd, b.pages, page, 0)
    nb, keep = batch_of(jn, b)
    q, k, v = (torch.randn(b.tokens, n, hd, device="cuda") for n in (heads, kv, kv))
    rope, out = jn.Rope(hd), torch.empty_like(q)
    cache.append_dev(1, nb, rope, heads, q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr())
    cache.append_dev(1, nb, rope, heads, q.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr())
    assert torch.equal(q, out)
    pools = [torch.randn(3, 5, kv, page, hd, device="cuda") for _ in range(2)]
    was = [p.clone() for p in pools]
    wrapped = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), 3, kv, hd, 5, page, 0)
    wrapped.copy_page_dev(4, 1)
    torch.cuda.synchronize()
    for p, w in zip(pools, was):
        w[:, 1] = w[:, 4]
        assert torch.equal(p, w)


# ---------------------------------------------------------------------------------------------- attention

def run_attention(jn, b, q, pools, half, scale, layer=0, y=None, check_workspace=True):
    heads, hd = q.shape[1], q.shape[2]
    layers, pages, kv, page, _ = pools[0].shape
    cache = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), layers, kv, hd, pages, page, 1 if half else 0)
    nb, keep = batch_of(jn, b)
    y = torch.full(q.shape, 7.0, device="cuda") if y is None else y
    n = cache.attention_workspace(nb, heads)
    ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")  # (what a workspace holds before is nobody's)
    cache.attention_dev(layer, nb, heads, q.data_ptr(), scale, y.data_ptr(), ws.data_ptr() if n else 0, n)
    torch.cuda.synchronize()
    return y


def check_rows(b, got, want, bound, skip=()):
    rows = [r for r, s, p in b.places() if s not in skip]
    err = np.abs(got[rows] - want[rows])
    assert (err <= bound[rows][:, :, None]).all(), (err.max(), bound[rows].min())
    # as a whole: a score's error is about 2^-24 of the largest scores (8), hence 2^-21 in a weight, the sums add less: 2^-19 with a factor of two over all
    assert np.linalg.norm(err) <= 2.0 ** -19 * np.linalg.norm(want[rows]) + 1e-30


SHAPES = [
    # hd, heads, kv, page, counts, lens, shared
    (64, 8, 2, 16, [1], [1], 0),
    (64, 8, 2, 16, [1], [600], 0),
    (128, 32, 8, 64, [1] * 9, [1, 2, 15, 16, 17, 31, 33, 64, 65], 0),
    (128, 7, 7, 32, [1, 1, 1], [1000, 3, 257], 0),
    (128, 16, 2, 16, [5, 1, 3, 0, 2], [500, 992, 1009, 0, 993], 61),       # shared pages end inside a step of 32; a sequence ends inside them
    (64, 14, 2, 128, [1] * 30, list(range(1025, 1055)), 8),
    (128, 40, 8, 32, [3] * 11, [700 + 31 * i for i in range(11)], 20),
    (192, 6, 2, 16, [2, 4], [300, 70], 0),
    (192, 6, 3, 32, [1] * 20, [200 + i for i in range(20)], 5),
    (256, 4, 1, 64, [1, 9], [130, 400], 1),
    (256, 8, 8, 256, [1, 1], [513, 700], 2),
    (64, 4, 4, 16, [70], [70], 0),                                        # a prompt: every row sees another length
    (128, 8, 2, 64, [130, 1], [300, 299], 0),
    (128, 71, 1, 16, [1, 2], [90, 45], 0),                                # one key/value head for 71 query heads
    (64, 2, 2, 16, [40] * 3, [3000, 60, 1200], 3),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,page,counts,lens,shared", SHAPES)
def test_attention(jn, half, hd, heads, kv, page, counts, lens, shared):
    rng = np.random.default_rng(hd + heads + len(counts))
    b = ref.Batch(rng, counts, lens, page, shared, pad_rows=2)
    g = torch.Generator(device="cuda").manual_seed(7)
    kind = torch.float16 if half else torch.float32
    pools = [torch.randn(2, b.pages, kv, page, hd, device="cuda", generator=g).to(kind) for _ in range(2)]
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    scale = 1 / np.sqrt(hd)
    got = run_attention(jn, b, q, pools, half, scale, layer=1)
    assert (got[b.starts[-1]:] == 7).all()  # rows behind the last sequence
    want, bound = ref.attention(q.cpu().numpy(), pools[0][1].cpu().numpy(), pools[1][1].cpu().numpy(), b, scale)
    check_rows(b, got.double().cpu().numpy(), want, bound)
    assert torch.equal(run_attention(jn, b, q, pools, half, scale, layer=1), got)  # and again, to the bit


PROMPTS = [
    # hd, heads, kv, page, counts, lens, shared: many rows, some of which see all and some almost nothing
    (64, 8, 4, 16, [130, 70, 200, 33, 90], [130, 75, 200, 33, 96], 0),
    (128, 12, 4, 64, [150, 0, 149, 151, 80], [150, 0, 300, 120, 333], 0),   # (one has rows in front of its first position)
    (128, 16, 2, 32, [300, 280], [900, 700], 0),                             # few spans of many rows
    (256, 12, 3, 128, [60, 70, 41], [60, 77, 300], 0),
    (192, 4, 2, 16, [129], [700], 0),
    (64, 16, 2, 64, [65, 140], [400, 350], 3),
    (64, 5, 1, 16, [90], [90], 0),                                           # fewer units of work than XCDs
    (128, 8, 1, 32, [40, 24, 11], [120, 500, 90], 2),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,heads,kv,page,counts,lens,shared", PROMPTS)
def test_attention_of_prompts(jn, half, hd, heads, kv, page, counts, lens, shared):
    test_attention(jn, half, hd, heads, kv, page, counts, lens, shared)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,shared", [(128, 0), (128, 4), (64, 2), (256, 1)])
def test_attention_ignores_what_a_row_does_not_see(jn, half, hd, shared):
    """NaN and infinities in the rest of the pages, on pages of nobody and in later tokens of the same pass; positions below 0; a lens of 0."""
    rng = np.random.default_rng(3)
    heads, kv, page = 8, 2, 32
    # (the fourth sequence has rows at positions -2 .. 1, the fifth has rows but no positions)
    b = ref.Batch(rng, [4, 1, 6, 4, 2, 1], [shared * page + 45, shared * page + 1, shared * page + 70, 2, 0, shared * page + 33], page, shared)
    g = torch.Generator(device="cuda").manual_seed(1)
    clean = [torch.randn(1, b.pages, kv, page, hd, device="cuda", generator=g).to(torch.float16 if half else torch.float32) for _ in range(2)]
    seen = np.zeros((b.pages, page), dtype=bool)
    for s, n in enumerate(b.lens):
        for p in range(n):
            seen[b.tables[s, p // page], p % page] = True
    hide = torch.from_numpy(~seen).cuda()[None, :, None, :, None]
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda")
    dirty = [torch.where(hide, bad[torch.randint(0, 3, c.shape, device="cuda", generator=g)].to(c.dtype), c) for c in clean]
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    want = run_attention(jn, b, q, clean, half, 0.1)
    got = run_attention(jn, b, q, dirty, half, 0.1)
    assert torch.equal(got, want) and torch.isfinite(got).all()
    exact, bound = ref.attention(q.cpu().numpy(), clean[0][0].cpu().numpy(), clean[1][0].cpu().numpy(), b, 0.1)
    check_rows(b, got.double().cpu().numpy(), exact, bound)
    blind = [r for r, s, p in b.places() if p < 0]
    assert len(blind) == 4 and (got[blind] == 0).all()
    # the last token of the third sequence, seen by its own row alone: keys and values of every kind there reach no other row
    s, pos = 2, b.lens[2] - 1
    for which in (0, 1):
        for value in (float("nan"), float("inf")):
            later = [c.clone() for c in clean]
            later[which][0, int(b.tables[s, pos // page]), :, pos % page] = value
            out = run_attention(jn, b, q, later, half, 0.1)
            own = int(b.starts[s + 1]) - 1
            others = [r for r in range(b.tokens) if r != own]
            assert torch.equal(out[others], want[others])
            assert torch.isnan(out[own]).all()


@pytest.mark.parametrize("half", [False, True])
def test_attention_of_bad_pages_and_lengths(jn, half):
    """A page that the cache does not have makes NaN of the rows that would have seen it and of no other; so does a lens beyond max_len."""
    rng = np.random.default_rng(4)
    hd, heads, kv, page, shared = 64, 4, 2, 16, 3
    b = ref.Batch(rng, [3, 2, 1, 4], [200, 190, 120, 100], page, shared)
    g = torch.Generator(device="cuda").manual_seed(2)
    pools = [torch.randn(1, b.pages, kv, page, hd, device="cuda", generator=g).to(torch.float16 if half else torch.float32) for _ in range(2)]
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    want = run_attention(jn, b, q, pools, half, 0.125)
    for page_id in (b.pages, -1, 1 << 30, -(1 << 31)):
        keep = b.tables.copy()
        b.tables[1, 150 // page] = page_id                # seen by both rows of sequence 1
        b.tables[3, 99 // page] = page_id                 # position 96 on: the rows at 96 .. 99, all four
        b.tables[0, 199 // page] = page_id                # position 192 on: all three rows of sequence 0
        got = run_attention(jn, b, q, pools, half, 0.125)
        nan = torch.isnan(got).all(dim=2).all(dim=1).cpu().numpy()
        assert list(nan) == [True] * 5 + [False] + [True] * 4
        assert torch.equal(got[5], want[5])
        b.tables[:] = keep
        b.lens[3] = 98                                    # rows at 94 .. 97: the first two do not reach position 96
        base = run_attention(jn, b, q, pools, half, 0.125)
        b.tables[3, 96 // page] = page_id
        got = run_attention(jn, b, q, pools, half, 0.125)
        assert torch.isnan(got[8:10]).all() and torch.equal(got[:8], base[:8])
        b.tables[:] = keep
        b.tables[0, 1] = page_id                          # a shared one: everybody
        assert torch.isnan(run_attention(jn, b, q, pools, half, 0.125)).all()
        b.tables[:] = keep
        b.lens[3] = 100
    b.lens[2] = 201                                       # max_len is 200
    got = run_attention(jn, b, q, pools, half, 0.125)
    assert torch.isnan(got[5]).all() and torch.equal(got[:5], want[:5]) and torch.equal(got[6:], want[6:])


@pytest.mark.parametrize("half", [False, True])
def test_attention_of_extreme_queries_and_scores(jn, half):
    """Queries far outside FP16, one key that takes all the weight among thousands, scores of equal weight, a negative and a zero scale."""
    rng = np.random.default_rng(6)
    hd, heads, kv, page = 128, 8, 2, 64
    b = ref.Batch(rng, [1, 1, 2, 1], [5000, 64, 1000, 700], page)
    g = torch.Generator(device="cuda").manual_seed(3)
    kind = torch.float16 if half else torch.float32
    pools = [torch.randn(1, b.pages, kv, page, hd, device="cuda", generator=g).to(kind) for _ in range(2)]
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    q[1] *= 1e6
    q[2] *= 1e-30
    q[3] = 0
    for scale in (1 / np.sqrt(hd), -0.05, 0.0):
        got = run_attention(jn, b, q, pools, half, scale).double().cpu().numpy()
        want, bound = ref.attention(q.cpu().numpy(), pools[0][0].cpu().numpy(), pools[1][0].cpu().numpy(), b, scale)
        err = np.abs(got - want)
        rows = [0, 2, 3, 4]
        assert (err[rows] <= bound[rows][:, :, None]).all()
        # row 1: scores of 10^6 and more, where one key is all; its value comes out as it is
        if scale != 0.0:
            assert np.abs(got[1] - want[1]).max() <= 2.0 ** -20 * 8


@pytest.mark.parametrize("half", [False, True])
def test_attention_with_offsets_past_32_bits(jn, half):
    """Pages at the far end of a pool of more than 4 GiB of keys."""
    hd, heads, kv, page = 64, 4, 1, 256
    pages = (9 << 30) // 2 // (kv * page * hd * (2 if half else 4))
    kind = torch.float16 if half else torch.float32
    pools = [torch.empty(1, pages, kv, page, hd, device="cuda", dtype=kind) for _ in range(2)]
    rng = np.random.default_rng(8)
    b = ref.Batch(rng, [1, 3], [700, 1000], page, 1, pages=16)
    b.tables = (b.tables + (pages - 16)).astype(np.int32)
    b.pages = pages
    g = torch.Generator(device="cuda").manual_seed(4)
    small = []
    for p in pools:
        p[0, pages - 16:] = torch.randn(16, kv, page, hd, device="cuda", generator=g).to(kind)
        small.append(p[0, pages - 16:].cpu().numpy())
    q = torch.randn(b.tokens, heads, hd, device="cuda", generator=g)
    got = run_attention(jn, b, q, pools, half, 0.125).double().cpu().numpy()
    b.tables = (b.tables - (pages - 16)).astype(np.int32)
    want, bound = ref.attention(q.cpu().numpy(), small[0], small[1], b, 0.125)
    check_rows(b, got, want, bound)
    # and an append there
    x = torch.randn(b.tokens, 2 * kv, hd, device="cuda", generator=g)
    b.tables = (b.tables + (pages - 16)).astype(np.int32)
    cache = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), 1, kv, hd, pages, page, 1 if half else 0)
    nb, keep = batch_of(jn, b)
    cache.append_dev(0, nb, None, 0, 0, 0, x.data_ptr(), x.data_ptr() + 4 * hd, k_stride=2 * hd, v_stride=2 * hd)
    for r, s, p in b.places():
        assert torch.equal(pools[0][0, int(b.tables[s, p // page]), :, p % page], x[r, :1].to(kind))
        assert torch.equal(pools[1][0, int(b.tables[s, p // page]), :, p % page], x[r, 1:].to(kind))


def test_recorded_pass_follows_its_arrays(jn):
    """Append and attention recorded once, replayed while lens, tables and inputs change and eager work of another batch runs in between, on another stream; every
    replay against an eager pass."""
    rng = np.random.default_rng(9)
    hd, heads, kv, page, shared = 128, 8, 2, 16, 5
    b = ref.Batch(rng, [2, 1, 3], [100, 90, 140], page, shared, max_len=300)
    nb, keep = batch_of(jn, b)
    pools = [torch.randn(1, b.pages, kv, page, hd, device="cuda").half() for _ in range(2)]
    cache = jn.PagedCache.wrap_dev(pools[0].data_ptr(), pools[1].data_ptr(), 1, kv, hd, b.pages, page, 1)
    rope = jn.Rope(hd)
    qkv, q, y = torch.randn(b.tokens, heads + 2 * kv, hd, device="cuda"), torch.empty(b.tokens, heads, hd, device="cuda"), torch.empty(b.tokens, heads, hd, device="cuda")
    ws = torch.empty(cache.attention_workspace(nb, heads), dtype=torch.uint8, device="cuda")
    row = (heads + 2 * kv) * hd
    other = torch.empty_like(y), torch.empty_like(ws)

    def both(out, space, stream):
        st = stream.cuda_stream
        cache.append_dev(0, nb, rope, heads, qkv.data_ptr(), q.data_ptr(), qkv.data_ptr() + 4 * heads * hd, qkv.data_ptr() + 4 * (heads + kv) * hd, row, 0, row, row, st)
        cache.attention_dev(0, nb, heads, q.data_ptr(), 0.1, out.data_ptr(), space.data_ptr(), space.numel(), stream_ptr=st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        both(y, ws, side)
    for i in range(4):
        qkv.normal_()
        keep[2].copy_(torch.tensor([100 + 50 * i, 90 + i, 140 - 20 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mine = pools[0].clone()
        both(other[0], other[1], torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(y, other[0]) and torch.equal(pools[0], mine) and torch.isfinite(y).all()


def test_serving_refusals_of_sizes(jn):
    from jitnn_amd import _lib
    b = ref.Batch(np.random.default_rng(0), [1], [6000], 16)
    cache = jn.PagedCache(1, 2, 64, b.pages, 16, 1)
    nb, keep = batch_of(jn, b)
    x = torch.zeros(4096, device="cuda")
    n = cache.attention_workspace(nb, 4)
    assert n > 0
    call = _lib.lib.jitnn_hip_paged_attention_dev
    p = x.data_ptr()
    assert call(cache.handle, 0, nb, 4, p, 256, 0.1, p, 256, p, n - 1, None) == _lib.EINVAL and "workspace" in _lib.last_error()
    assert call(cache.handle, 0, nb, 4, p, 256, 0.1, p, 256, None, n, None) == _lib.EINVAL
    assert call(cache.handle, 0, nb, 4, p, 256, 0.1, p, 256, p + 4, 1 << 30, None) == _lib.EINVAL
    with pytest.raises(ValueError, match="aligned|multiple"):
        jn.PagedCache.wrap_dev(p + 4, p, 1, 2, 64, 1, 16, 1)
    rope = jn.Rope(12)
    with pytest.raises(jn.UnsupportedTypeError, match="multiple of 8"):
        cache.append_dev(0, nb, rope, 0, 0, 0, p, p)
    with pytest.raises(ValueError, match="rot_dim"):
        cache.append_dev(0, nb, jn.Rope(128), 0, 0, 0, p, p)


# ---------------------------------------------------------------------------------------------- drafted tokens

def run_verify(jn, logits, starts, tokens, q, temps, uniforms, stride=0, rows_of_call=None):
    rows, vocab = logits.shape
    wide = np.zeros((rows, vocab + stride), dtype=np.float32)
    wide[:, :vocab] = logits
    keep = [dev(wide), dev(np.asarray(starts, np.int32)), dev(np.asarray(tokens, np.int32)), dev(np.asarray(temps, np.float32)), dev(np.asarray(uniforms, np.float32))]
    dq = None
    if q is not None:
        wq = np.zeros((rows, vocab + 2 * stride), dtype=np.float32)
        wq[:, :vocab] = q
        dq = dev(wq)
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    acc = torch.full((len(temps),), -7, dtype=torch.int32, device="cuda")
    rows = rows if rows_of_call is None else rows_of_call
    n = jn.verify_workspace(rows, len(temps), vocab)
    ws = torch.full((n // 4 + 4,), float("nan"), device="cuda")
    jn.verify_drafts_dev(keep[0].data_ptr(), rows, vocab, keep[1].data_ptr(), len(temps), keep[2].data_ptr(), keep[3].data_ptr(), keep[4].data_ptr(), out.data_ptr(),
                         acc.data_ptr(), ws.data_ptr(), n, 0 if dq is None else dq.data_ptr(), vocab + stride, vocab + 2 * stride)
    torch.cuda.synchronize()
    return out.cpu().numpy(), acc.cpu().numpy()


def drafts(rng, counts, vocab, spread=3.0, near=0.5):
    rows = sum(counts) + 2  # two behind the last sequence
    logits = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    temps = [0.0 if i % 3 == 2 else float(np.float32(0.5 + 0.3 * (i % 4))) for i in range(len(counts))]
    starts = np.concatenate([[0], np.cumsum(counts)])
    q = np.zeros((rows, vocab), dtype=np.float32)
    tokens = rng.integers(0, vocab, rows)
    for s, c in enumerate(counts):
        for r in range(starts[s], starts[s] + c):
            z = (logits[r].astype(np.float64) + near * rng.standard_normal(vocab)) / (temps[s] or 1.0)
            w = np.exp(z - z.max())
            q[r] = (w / w.sum()).astype(np.float32)
            if r + 1 < starts[s] + c:
                tokens[r + 1] = rng.choice(vocab, p=w / w.sum())
    return logits, starts, tokens, q, temps, rng.random((rows, 2)).astype(np.float32)


@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("counts,vocab,stride", [([1], 1, 0), ([5], 50, 0), ([3, 1, 9, 0, 2, 6], 1000, 0), ([4] * 11, 8192, 1), ([2, 7, 7], 8193, 3), ([5, 3, 4], 32000, 0),
                                                 ([9, 2, 1, 4], 128256, 0), ([3, 3], 600001, 0)])
def test_verify(jn, with_q, counts, vocab, stride):
    rng = np.random.default_rng(vocab)
    for round_ in range(4):
        logits, starts, tokens, q, temps, u = drafts(rng, counts, vocab, near=(0.0, 0.1, 0.5, 2.0)[round_])
        q = q if with_q else None
        want = ref.verify(logits, starts, tokens, q, temps, u)
        got = run_verify(jn, logits, starts, tokens, q, temps, u, stride)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


@pytest.mark.parametrize("vocab", [20000, 9000])  # (of few chunks the draw sums by itself what a draft left)
@pytest.mark.parametrize("with_q", [False, True])
def test_verify_of_odd_logits_and_numbers(jn, with_q, vocab):
    """Equal largest logits, NaN and infinities, rows of nothing else, random numbers of 0 and just below 1, drafts that are no tokens or have no probability."""
    rng = np.random.default_rng(1)
    counts = [4] * 12
    logits, starts, tokens, q, temps, u = drafts(rng, counts, vocab)
    temps = [0.0, 1.0, 0.7] * 4
    below_one = np.float32(1 - 2.0 ** -24)
    u[0:8] = 0
    u[8:16] = below_one
    logits[1, [500, 8192, vocab - 1]] = logits[1].max() + 1                     # equal largest ones, in three chunks
    logits[4:8, ::2] = np.nan
    logits[5, 1::2] = -np.inf                                              # nothing at all
    logits[9, 7777] = np.inf
    logits[13, [3, 8345]] = np.inf                                        # two that share all the weight
    logits[17] = -np.inf
    logits[18] = np.nan
    logits[19, :vocab - 1000] = -np.inf
    tokens[21], tokens[22], tokens[25], tokens[26] = vocab, -1, 1 << 30, -(1 << 31)
    q[28, tokens[29]] = 0
    logits[32, tokens[33]] = -np.inf
    tokens[37] = int(np.argmax(logits[36]))
    temps[9] = float("nan")                                                # as 0: greedy
    want = ref.verify(logits, starts, tokens, q if with_q else None, [0.0 if not t > 0 else t for t in temps], u)
    got = run_verify(jn, logits, starts, tokens, q if with_q else None, temps, u)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0]), (np.argwhere(got[0] != want[0]), got[0], want[0])


def test_verify_of_no_rows(jn):
    """Sequences without rows, with and without draft probabilities: nothing kept, and nothing else written."""
    for q in (None, np.zeros((1, 9000), np.float32)):
        out, acc = run_verify(jn, np.zeros((1, 9000), np.float32), [0, 0, 0], [0], q, [1.0, 0.0], np.zeros((1, 2), np.float32), rows_of_call=0)
        assert list(acc) == [0, 0] and list(out) == [-7]


def test_verify_follows_the_target(jn):
    """One draft per sequence, drawn from another distribution: the first emitted token is distributed as the target's p (chi-squared over 65280 sequences, 49 degrees of
    freedom: mean 49, standard deviation 9.9; five of those above)."""
    rng = np.random.default_rng(2)
    vocab, n = 50, 32640
    base = (1.5 * rng.standard_normal(vocab)).astype(np.float32)
    zq = base + rng.standard_normal(vocab)
    qp = np.exp(zq - zq.max())
    qp /= qp.sum()
    p = np.exp(base.astype(np.float64) - base.max())
    p /= p.sum()
    count = np.zeros(vocab)
    for _ in range(2):
        starts, tokens = np.arange(0, 2 * n + 2, 2), np.zeros(2 * n, dtype=np.int32)
        tokens[1::2] = rng.choice(vocab, size=n, p=qp)
        out, acc = run_verify(jn, np.tile(base, (2 * n, 1)), starts, tokens, np.tile(qp.astype(np.float32), (2 * n, 1)), np.ones(n, np.float32), rng.random((2 * n, 2)))
        assert set(acc) == {0, 1}
        count += np.bincount(out[0::2], minlength=vocab)
    chi = ((count - 2 * n * p) ** 2 / (2 * n * p)).sum()
    assert chi <= 49 + 5 * 9.9


def test_verify_refusals(jn):
    from jitnn_amd import _lib
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    call = _lib.lib.jitnn_hip_verify_drafts_dev
    n = jn.verify_workspace(2, 1, 100)
    ok = [p, 100, 2, 100, p, 1, p, None, 0, p, p, p, p, p, n, None]
    for at, bad in ((0, None), (1, 99), (2, -1), (2, 65536), (3, 0), (4, None), (5, -1), (6, None), (9, None), (10, None), (11, None), (12, None), (13, None), (14, n - 1)):
        args = list(ok)
        args[at] = bad
        assert call(*args) == _lib.EINVAL, at
    args = list(ok)
    args[7], args[8] = p, 99
    assert call(*args) == _lib.EINVAL
    args = list(ok)
    args[5] = 0
    assert call(*args) == 0
