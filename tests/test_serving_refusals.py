"""What the operators of a served batch refuse, and the host side of drafting: no device needed."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    from jitnn_amd import _lib
    return _lib


def wrap(lib, layers=2, kv=2, hd=64, pages=3, page=16, kind=1, k=1 << 20, v=1 << 21):
    h = C.c_void_p()
    return lib.lib.jitnn_hip_paged_cache_wrap_dev(k, v, layers, kv, hd, pages, page, kind, C.byref(h)), h


def test_cache_shapes(lib):
    size = lib.lib.jitnn_hip_paged_cache_nbytes
    assert size(2, 3, 128, 5, 64, 1) == 2 * 3 * 128 * 5 * 64 * 2 and size(2, 3, 128, 5, 64, 0) == 2 * 3 * 128 * 5 * 64 * 4
    assert size(1, 1, 256, 1 << 20, 256, 0) == 1 << 38
    for bad in ((0, 1, 64, 1, 16, 1), (1, 0, 64, 1, 16, 1), (1, 1, 80, 1, 16, 1), (1, 1, 64, 0, 16, 1), (1, 1, 64, 1, 8, 1), (1, 1, 64, 1, 48, 1), (1, 1, 64, 1, 512, 1),
                (1, 1, 64, 1, 16, 2), (1, 1, 64, 1, 16, 30), (1 << 20, 65535, 256, 1 << 30, 256, 0)):
        assert size(*bad) == lib.EINVAL, bad
    for bad in (dict(hd=65), dict(page=0), dict(k=None), dict(v=1 << 21 | 4), dict(kind=8)):
        rc, h = wrap(lib, **bad)
        assert rc == lib.EINVAL and h.value is None, bad
    assert lib.lib.jitnn_hip_paged_cache_free(None) == 0 and lib.lib.jitnn_hip_rope_free(None) == 0


def test_batches_and_arguments(lib):
    from jitnn_amd import Batch
    rc, h = wrap(lib)
    assert rc == 0
    p, row = 1 << 22, 2 * 64
    good = dict(sequences=2, tokens=3, max_tokens=2, max_len=48, tables_ptr=p, table_stride=3, starts_ptr=p, lens_ptr=p, shared_pages=1)

    def append(batch, layer=0, heads=4, **kw):
        a = dict(q=p, qs=4 * 64, qo=p, qos=4 * 64, k=p, ks=row, v=p, vs=row)
        a.update(kw)
        return lib.lib.jitnn_hip_paged_append_dev(h, layer, batch, None, a["q"], a["qs"], heads, a["qo"], a["qos"], a["k"], a["ks"], a["v"], a["vs"], None)

    def attend(batch, layer=0, heads=4, **kw):
        a = dict(q=p, qs=heads * 64, scale=0.1, y=p, ys=heads * 64)
        a.update(kw)
        return lib.lib.jitnn_hip_paged_attention_dev(h, layer, batch, heads, a["q"], a["qs"], a["scale"], a["y"], a["ys"], None, 0, None)

    for bad in (dict(sequences=-1), dict(tokens=-1), dict(max_tokens=-1), dict(max_len=-1), dict(max_len=49), dict(shared_pages=4), dict(shared_pages=-1), dict(table_stride=-1),
                dict(tables_ptr=0), dict(starts_ptr=0), dict(lens_ptr=0), dict(sequences=65536), dict(max_len=(1 << 30) + 1, table_stride=1 << 27)):
        b = Batch(**{**good, **bad})
        assert append(b) == lib.EINVAL and attend(b) == lib.EINVAL, bad
        assert lib.lib.jitnn_hip_paged_attention_workspace(h, b, 4) == lib.EINVAL
    b = Batch(**good)
    for call in (append, attend):
        assert call(b, layer=2) == lib.EINVAL and call(b, layer=-1) == lib.EINVAL and call(None) == lib.EINVAL
    for bad in (dict(heads=-1), dict(k=None), dict(v=None), dict(q=None), dict(qo=None), dict(ks=row - 1), dict(vs=4), dict(qs=8), dict(qos=4 * 64 + 4)):
        assert append(b, **bad) == lib.EINVAL, bad
    for bad in (dict(k=p + 4), dict(ks=row + 2), dict(qo=p + 8)):
        assert append(b, **bad) == lib.EUNSUPPORTED, bad
    for bad in (dict(heads=0), dict(heads=3), dict(q=None), dict(y=None), dict(qs=8), dict(ys=255), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attend(b, **bad) == lib.EINVAL, bad
    # nothing to do: no device, no arrays
    for empty in (dict(tokens=0), dict(sequences=0)):
        b = Batch(**{**good, **empty, "tables_ptr": 0, "starts_ptr": 0, "lens_ptr": 0})
        assert append(b) == 0 and attend(b) == 0 and lib.lib.jitnn_hip_paged_attention_workspace(h, b, 4) == 0
    copy = lib.lib.jitnn_hip_paged_cache_copy_page_dev
    assert copy(h, 3, 0, None) == lib.EINVAL and copy(h, 0, -1, None) == lib.EINVAL and copy(h, 1, 1, None) == 0 and copy(None, 0, 0, None) == lib.EINVAL
    assert lib.lib.jitnn_hip_paged_cache_free(h) == 0


def test_null_handles(lib):
    from jitnn_amd import Batch
    b = Batch(1, 1, 1, 1, 16, 1, 16, 16)
    assert lib.lib.jitnn_hip_paged_append_dev(None, 0, b, None, None, 0, 0, None, 0, None, 0, None, 0, None) == lib.EINVAL
    assert lib.lib.jitnn_hip_paged_attention_dev(None, 0, b, 1, None, 0, 1.0, None, 0, None, 0, None) == lib.EINVAL
    assert lib.lib.jitnn_hip_llama_step_dev(None, None, b, None, None, 0, None, None) == lib.EINVAL
    assert lib.lib.jitnn_hip_llama_set_rope(None, None) == lib.EINVAL
    h = C.c_void_p(1)
    create = lib.lib.jitnn_hip_rope_create
    for bad in ((3, 0, 1e4), (0, 0, 1e4), (1026, 0, 1e4), (64, 0, 0.0), (64, 0, -1.0), (64, 0, float("inf"))):
        assert create(*bad, None, None, C.byref(h)) == lib.EINVAL and h.value is None, bad
    assert create(64, 0, 1e4, None, None, None) == lib.EINVAL


def test_workspace_of_drafts(lib):
    n = lib.lib.jitnn_hip_verify_workspace
    assert n(1, 1, 1) == 24 and n(5, 2, 4096) == 96 and n(5, 2, 4097) == 192
    assert n(-1, 1, 1) == lib.EINVAL and n(1, -1, 1) == lib.EINVAL and n(1, 1, 0) == lib.EINVAL and n(65536, 1, 10) == lib.EINVAL
    assert n(1, 1, (1 << 30) + 1) == lib.EINVAL and n(1, 1, 1 << 30) == (24 + 8 - 8) * (1 << 18) and n(0, 3, 1) == 24


def test_requests_with_drafts():
    from jitnn_amd import GenerationRequest
    assert GenerationRequest("p", draft_tokens=3).draft_tokens == 3 and GenerationRequest("p").draft_tokens == 0
    assert GenerationRequest("p", temperature=0.7, top_k=1, draft_tokens=3).draft_tokens == 3
    for bad in (dict(draft_tokens=-1), dict(draft_tokens=2, temperature=0.5, top_k=40), dict(draft_tokens=2, temperature=0.5, top_p=0.9)):
        with pytest.raises(ValueError):
            GenerationRequest("p", **bad)


def test_drafts_are_looked_up_where_the_last_tokens_stood_before():
    from jitnn_amd.llm import look_up_draft
    assert look_up_draft([], 4) == [] and look_up_draft([7], 4) == [] and look_up_draft([7, 8, 9], 4) == []
    assert look_up_draft([1, 2, 3, 4, 1, 2], 4) == [3, 4, 1, 2]
    assert look_up_draft([1, 2, 3, 4, 1, 2], 1) == [3]
    assert look_up_draft([1, 2, 5, 1, 2, 6, 1, 2], 2) == [6, 1]        # the last place
    assert look_up_draft([9, 2, 6, 1, 2], 3) == [6, 1, 2]              # one token where two did not stand before
    assert look_up_draft([4, 4], 3) == [4] and look_up_draft([4, 4, 4], 3) == [4]


def test_reference_verification_keeps_what_it_must():
    """The oracle of the GPU tests by hand: p = (1/2, 1/4, 1/4), a draft kept below its share and not at it, the rest without it."""
    import serving_reference as ref
    logits = np.log(np.array([[2, 1, 1], [1, 1, 2]], dtype=np.float64)).astype(np.float32)
    for u, want in ((0.49, ([0, 2], 1)), (0.51, ([1, -1], 0))):
        out, acc = ref.verify(logits, [0, 2], [5, 0], None, [1.0], [[u, 0.2], [0.3, 0.9]])
        assert list(out) == want[0] and list(acc) == [want[1]]
