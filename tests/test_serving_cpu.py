"""What the serving operators refuse on the host, through the C ABI and through the torch view: no GPU is needed, and nothing is launched."""
import ctypes as C

import pytest
import torch

P = 1 << 20                                            # a 16-byte aligned address that is never read


def cache(K, **change):
    c = K.KvCache()
    c.dtype, c.head_dim, c.n_kv_heads, c.page_size, c.n_pages, c.k, c.v = K.KV_BF16, 64, 2, 16, 8, P, P
    c.page_stride, c.head_stride, c.row_stride = 2 * 16 * 64, 16 * 64, 64
    c.scale_page_stride, c.scale_head_stride, c.scale_row_stride = 32, 16, 1
    for k, v in change.items():
        setattr(c, k, v)
    return c


def batch(K, **change):
    b = K.KvBatch()
    b.n_seqs, b.max_pages, b.q_start, b.kv_len, b.pages, b.pages_stride = 2, 4, P, P, P, 4
    for k, v in change.items():
        setattr(b, k, v)
    return b


def attention_args(K, **change):
    a = K.PagedAttentionArgs()
    a.n_rows, a.n_heads, a.q, a.out, a.scale, a.causal = 3, 4, P, P, 0.125, 1
    a.q_row_stride = a.out_row_stride = 256
    a.q_head_stride = a.out_head_stride = 64
    for k, v in change.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [({"dtype": 2}, "dtype"), ({"head_dim": 96}, "head_dim"), ({"n_kv_heads": 0}, "n_kv_heads"), ({"page_size": 0}, "page_size"), ({"n_pages": -1}, "n_pages"),
             ({"k": None}, "null"), ({"k": P + 8}, "16-byte"), ({"row_stride": 68}, "16-byte"), ({"head_stride": -8}, "negative"), ({"dtype": 1}, "scales"),
             ({"dtype": 1, "row_stride": 72, "k_scale": P, "v_scale": P}, "16-byte")]
BAD_BATCH = [({"n_seqs": -1}, "negative"), ({"max_pages": -1}, "negative"), ({"q_start": None}, "null"), ({"pages": None}, "null"), ({"kv_len": P + 2}, "misaligned"),
             ({"status": P + 1}, "misaligned"), ({"max_new": -1}, "negative")]


@pytest.mark.parametrize("change,say", BAD_CACHE + [(None, "null")])
def test_bad_caches(ofa, change, say):
    K, lib = ofa.capi, ofa.capi.load()
    c = C.byref(cache(K, **change)) if change is not None else None
    for rc in (lib.ofa_kv_append(c, C.byref(batch(K)), P, P, 3, 128, 64, 128, 64, None), lib.ofa_kv_read(c, C.byref(batch(K)), P, P, 3, 128, 64, 128, 64, None),
               lib.ofa_paged_attention(c, C.byref(batch(K)), C.byref(attention_args(K)), None)):
        assert rc == K.BAD_ARGUMENT and say in lib.ofa_serving_last_error().decode()
    assert lib.ofa_paged_attention_workspace(c, C.byref(batch(K)), 3, 4) == 0


@pytest.mark.parametrize("change,say", BAD_BATCH)
def test_bad_batches(ofa, change, say):
    K, lib = ofa.capi, ofa.capi.load()
    for rc in (lib.ofa_kv_append(C.byref(cache(K)), C.byref(batch(K, **change)), P, P, 3, 128, 64, 128, 64, None),
               lib.ofa_paged_attention(C.byref(cache(K)), C.byref(batch(K, **change)), C.byref(attention_args(K)), None)):
        assert rc == K.BAD_ARGUMENT and say in lib.ofa_serving_last_error().decode()


@pytest.mark.parametrize("args", [(None, P, 3, 128, 64, 128, 64), (P, P + 8, 3, 128, 64, 128, 64), (P, P, 3, 124, 64, 128, 64), (P, P, 3, 128, 64, 128, -64), (P, P, -1, 128, 64, 128, 64)])
def test_bad_rows(ofa, args):
    K, lib = ofa.capi, ofa.capi.load()
    for fn in (lib.ofa_kv_append, lib.ofa_kv_read):
        assert fn(C.byref(cache(K)), C.byref(batch(K)), *args, None) == K.BAD_ARGUMENT


@pytest.mark.parametrize("change,say", [({"n_heads": 3}, "multiple"), ({"n_heads": 0}, "multiple"), ({"n_rows": -1}, "negative"), ({"window": -1}, "window"), ({"window": 5, "causal": 0}, "window"),
                                        ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"q": None}, "q is null"), ({"out": None}, "out is null"),
                                        ({"q": P + 4}, "16-byte"), ({"out_row_stride": 252}, "16-byte"), ({"q_head_stride": -64}, "16-byte"), ({"lse": P + 2}, "lse"),
                                        ({"n_rows": 2 ** 31 - 1, "n_heads": 2 ** 16}, "too many"), ({"n_rows": 2 ** 30, "n_heads": 2 ** 16}, "too many")])
def test_bad_attention(ofa, change, say):
    K, lib = ofa.capi, ofa.capi.load()
    assert lib.ofa_paged_attention(C.byref(cache(K)), C.byref(batch(K)), C.byref(attention_args(K, **change)), None) == K.BAD_ARGUMENT
    assert say in lib.ofa_serving_last_error().decode()


def test_rows_that_overlap_where_they_are_written(ofa):
    K, lib = ofa.capi, ofa.capi.load()
    said = lambda: lib.ofa_serving_last_error().decode()  # noqa: E731
    for strides in ((0, 64, 128, 64), (128, 0, 128, 64), (128, 64, 64, 64), (128, 64, 128, 56), (128, 64, 64, 128)):
        assert lib.ofa_kv_read(C.byref(cache(K)), C.byref(batch(K)), P, P, 3, *strides, None) == K.BAD_ARGUMENT and "overlap" in said()
    for change in ({"row_stride": 0}, {"head_stride": 0}, {"page_stride": 0}, {"row_stride": 56}, {"head_stride": 64}, {"dtype": 1, "k_scale": P, "v_scale": P, "scale_row_stride": 0},
                   {"dtype": 1, "k_scale": P, "v_scale": P, "scale_page_stride": 16}):
        assert lib.ofa_kv_append(C.byref(cache(K, **change)), C.byref(batch(K)), P, P, 3, 128, 64, 128, 64, None) == K.BAD_ARGUMENT and "overlap" in said()
    for change in ({"out_row_stride": 0}, {"out_row_stride": 192}, {"out_head_stride": 0}, {"out_head_stride": 56}):
        assert lib.ofa_paged_attention(C.byref(cache(K)), C.byref(batch(K)), C.byref(attention_args(K, **change)), None) == K.BAD_ARGUMENT and "overlap" in said()


@pytest.mark.parametrize("rows,vocab,ins,outs,off", [(3, 100, 100, 100, 1), (3, 100, 100, 100, -1), (3, 100, 100, 100, 100), (3, 100, 200, 200, 99), (3, 100, 200, 200, 101),
                                                        (3, 100, 200, 100, 0), (3, 100, 100, 200, 0), (1, 100, 100, 100, 99), (3, 100, 0, 100, 0), (3, 100, 0, 100, 50)])
def test_logits_that_overlap(ofa, rows, vocab, ins, outs, off):
    """The calls that are allowed (in place, side by side in one tensor) run in the GPU's tests"""
    K, lib = ofa.capi, ofa.capi.load()
    a = K.LogitsArgs()
    a.dtype, a.n_rows, a.vocab, a.inp, a.out, a.in_stride, a.out_stride = K.DTYPE_F32, rows, vocab, P, P + off * 4, ins, outs
    assert lib.ofa_logits_process(C.byref(a), None) == K.BAD_ARGUMENT and "overlap" in lib.ofa_serving_last_error().decode()


def test_a_workspace_that_is_too_small(ofa):
    K, lib = ofa.capi, ofa.capi.load()
    c, b = cache(K, n_pages=4096), batch(K, max_pages=2048, max_new=1)
    need = lib.ofa_paged_attention_workspace(C.byref(c), C.byref(b), 3, 4)
    assert need > 0
    for w, n in ((None, need), (P, need - 1), (P + 4, need)):
        assert lib.ofa_paged_attention(C.byref(c), C.byref(b), C.byref(attention_args(K, workspace=w, workspace_bytes=n)), None) == K.BAD_ARGUMENT
        assert "workspace" in lib.ofa_serving_last_error().decode()


def test_empty_calls_launch_nothing(ofa):
    K, lib = ofa.capi, ofa.capi.load()
    c, b = cache(K), batch(K)
    assert lib.ofa_kv_append(C.byref(c), C.byref(b), None, None, 0, 0, 0, 0, 0, None) == K.OK
    assert lib.ofa_kv_read(C.byref(c), C.byref(batch(K, n_seqs=0, q_start=None, kv_len=None, pages=None)), None, None, 5, 0, 0, 0, 0, None) == K.OK
    assert lib.ofa_paged_attention(C.byref(c), C.byref(b), C.byref(attention_args(K, n_rows=0, q=None, out=None)), None) == K.OK
    a = K.LogitsArgs()
    assert lib.ofa_logits_process(C.byref(a), None) == K.OK


@pytest.mark.parametrize("change,say", [({"dtype": 7}, "dtype"), ({"n_rows": -1}, "negative"), ({"n_rows": 70000}, "65535"), ({"inp": None}, "null"), ({"out": P + 2}, "misaligned"),
                                        ({"out_stride": 50}, "overlap"), ({"in_stride": -100}, "negative"), ({"repetition": P, "max_tokens": 4}, "tokens"), ({"bias": P}, "together"),
                                        ({"mask": P + 1}, "misaligned"), ({"max_bias": -1}, "negative"), ({"vocab": 2 ** 30 + 1}, "2^30"), ({"tokens": P, "max_tokens": 2 ** 29 + 1}, "2^29")])
def test_bad_logits(ofa, change, say):
    K, lib = ofa.capi, ofa.capi.load()
    a = K.LogitsArgs()
    a.dtype, a.n_rows, a.vocab, a.inp, a.out, a.in_stride, a.out_stride = K.DTYPE_F32, 2, 100, P, P, 100, 100
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.ofa_logits_process(C.byref(a), None) == K.BAD_ARGUMENT and say in lib.ofa_serving_last_error().decode()
    assert lib.ofa_logits_process(None, None) == K.BAD_ARGUMENT


def test_structures_have_the_headers_sizes(ofa):
    """the ctypes mirror lays its fields out as the header does (natural alignment, 64-bit)"""
    K = ofa.capi
    assert (C.sizeof(K.KvCache), C.sizeof(K.KvBatch), C.sizeof(K.PagedAttentionArgs), C.sizeof(K.LogitsArgs)) == (104, 56, 96, 160)


def test_tensors_on_the_host_are_refused(ofa):
    sv = ofa.serving
    with pytest.raises(ofa.OfaError) as e:
        sv.KVCache(torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16))
    assert e.value.code == ofa.capi.BAD_ARGUMENT and "CUDA tensor" in str(e.value)
    with pytest.raises(ofa.OfaError):
        sv.KVBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32))
    for bad in (torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.float64), None):
        with pytest.raises(ofa.OfaError):
            sv.logits_process(bad)
    with pytest.raises(ofa.OfaError):
        sv.KVCache.empty(2, 16, 1, 64, "int8")
