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
