"""What else the serving operators refuse on the host, and how the extension beside them is built: no GPU is needed."""
import ctypes as C
import os

import torch

from test_serving_cpu import P, attention_args, batch, cache


def test_a_page_table_that_runs_backwards(ofa):
    K, lib = ofa.capi, ofa.capi.load()
    b = batch(K, pages_stride=-4)
    for rc in (lib.ofa_kv_append(C.byref(cache(K)), C.byref(b), P, P, 3, 128, 64, 128, 64, None), lib.ofa_kv_read(C.byref(cache(K)), C.byref(b), P, P, 3, 128, 64, 128, 64, None),
               lib.ofa_paged_attention(C.byref(cache(K)), C.byref(b), C.byref(attention_args(K)), None)):
        assert rc == K.BAD_ARGUMENT and "negative stride" in lib.ofa_serving_last_error().decode()
    assert lib.ofa_paged_attention_workspace(C.byref(cache(K)), C.byref(b), 3, 4) == 0


def test_the_extension_of_another_torch_is_not_taken(ofa, monkeypatch):
    """It looks at tensors in place: each torch has a file of its own"""
    sv, build = ofa.serving, ofa.build_mod
    path = build.build_host()
    assert path is None or torch.__version__ in os.path.basename(path) and sv._bind() is not None
    monkeypatch.setattr(torch, "__version__", "1.2.3+none")
    assert sv._bind() is None and not os.path.exists(build.host_path("1.2.3+none"))


def test_keys_and_values_upon_one_another(ofa):
    K, lib = ofa.capi, ofa.capi.load()
    said = lambda: lib.ofa_serving_last_error().decode()  # noqa: E731
    page = 2 * 16 * 64                                           # elements of a page of the helper's cache

    def append(**change):
        return lib.ofa_kv_append(C.byref(cache(K, **change)), C.byref(batch(K)), P, P, 3, 128, 64, 128, 64, None)
    scales = {"dtype": 1, "k": P, "v": P + (1 << 20), "k_scale": P, "v_scale": P}
    for change in ({"v": P}, {"v": P + 2 * page}, {"v": P + 2 * (8 * page - 64)}, {"k": P + 2 * page}, {"v": P + 2 * page, "page_stride": 2 * page - 64}, scales, dict(scales, v=P + page),
                   dict(scales, v_scale=P + 8 * 32 - 1)):
        assert append(**change) == K.BAD_ARGUMENT and "overlap" in said(), change
    for args in ((P, P), (P, P + 2 * 64), (P, P + 2 * 128 * 2), (P + 2 * 64, P)):
        assert lib.ofa_kv_read(C.byref(cache(K)), C.byref(batch(K)), *args, 3, 128, 64, 128, 64, None) == K.BAD_ARGUMENT and "overlap" in said(), args
    # beside one another they are fine: what is refused then is what comes behind that check
    assert lib.ofa_kv_append(C.byref(cache(K, n_pages=0, k=None, v=None)), C.byref(batch(K)), P, P, 0, 128, 64, 128, 64, None) == K.OK
