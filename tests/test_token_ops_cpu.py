"""Argument checks of the token-model operators: descriptor validation, workspace sizes and the Python wrappers'
refusals need no GPU. Every refused call returns before anything is launched."""
import ctypes

import pytest
import torch

import neuzephyr_b200 as nz
from neuzephyr_b200 import _capi as C

FAKE = 1 << 20  # an aligned address that no refused call follows


def _embedding(**kw):
    d = C.EmbeddingDesc(tokens=10, vocab=100, dim=64, ld_table=64, ld_y=64, padding_index=-1, scale=1.0, dtype=C.F16,
                        table_dtype=C.F32, index_type=C.I64, overwrite=1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", [
    (dict(tokens=-1), C.ERR_BAD_ARG), (dict(vocab=-1), C.ERR_BAD_ARG), (dict(dim=-1), C.ERR_BAD_ARG),
    (dict(ld_table=63), C.ERR_BAD_ARG), (dict(ld_y=63), C.ERR_BAD_ARG), (dict(dtype=3), C.ERR_BAD_ARG),
    (dict(table_dtype=-1), C.ERR_BAD_ARG), (dict(index_type=2), C.ERR_BAD_ARG), (dict(table_dtype=C.BF16), C.ERR_UNSUPPORTED),
    (dict(vocab=2 ** 31 - 1), C.ERR_UNSUPPORTED), (dict(tokens=2 ** 31), C.ERR_UNSUPPORTED),
])
def test_embedding_refusals(change, code):
    L = C.lib()
    d = _embedding(**change)
    assert L.nzb_embedding_forward(ctypes.byref(d), FAKE, FAKE, FAKE, None) == code
    assert L.nzb_last_error_string()


def test_embedding_pointers_and_workspace():
    L = C.lib()
    d, n = _embedding(), ctypes.c_size_t(0)
    assert L.nzb_embedding_forward(None, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_forward(ctypes.byref(d), None, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_forward(ctypes.byref(d), FAKE, None, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_forward(ctypes.byref(d), FAKE, FAKE, FAKE + 1, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_forward(ctypes.byref(d), FAKE + 2, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_forward(ctypes.byref(d), FAKE, FAKE + 4, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_backward_workspace_bytes(ctypes.byref(d), None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == C.OK and n.value > 0
    small = n.value
    assert L.nzb_embedding_backward(ctypes.byref(d), FAKE, FAKE, FAKE, None, 0, None) == C.ERR_WORKSPACE
    assert L.nzb_embedding_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, small - 1, None) == C.ERR_WORKSPACE
    assert L.nzb_embedding_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE + 16, small, None) == C.ERR_WORKSPACE
    assert L.nzb_embedding_backward(ctypes.byref(d), FAKE, FAKE, FAKE + 2, FAKE, small, None) == C.ERR_BAD_ARG
    assert L.nzb_embedding_backward(ctypes.byref(d), None, FAKE, FAKE, FAKE, small, None) == C.ERR_BAD_ARG
    d.tokens = 100000
    assert L.nzb_embedding_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == C.OK and n.value > small
    # nothing to do: no pointer is looked at
    d = _embedding(tokens=0, overwrite=0)
    assert L.nzb_embedding_forward(ctypes.byref(d), None, None, None, None) == C.OK
    assert L.nzb_embedding_backward(ctypes.byref(d), None, None, None, None, 0, None) == C.OK


def _layernorm(**kw):
    d = C.LayernormDesc(rows=7, dim=96, ld_x=96, ld_y=96, ld_dx=96, eps=1e-5, dtype=C.BF16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), C.ERR_BAD_ARG), (dict(dim=-2), C.ERR_BAD_ARG), (dict(ld_x=95), C.ERR_BAD_ARG), (dict(ld_y=95), C.ERR_BAD_ARG),
    (dict(dtype=7), C.ERR_BAD_ARG), (dict(eps=-1e-5), C.ERR_BAD_ARG), (dict(eps=float("nan")), C.ERR_BAD_ARG),
    (dict(dim=1 << 25, ld_x=1 << 25, ld_y=1 << 25), C.ERR_UNSUPPORTED),
])
def test_layernorm_refusals(change, code):
    L = C.lib()
    d = _layernorm(**change)
    assert L.nzb_layernorm_forward(ctypes.byref(d), FAKE, None, None, FAKE, None, None, None) == code
    assert L.nzb_layernorm_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == code


def test_layernorm_pointers():
    L = C.lib()
    d, n = _layernorm(), ctypes.c_size_t(0)
    assert L.nzb_layernorm_forward(ctypes.byref(d), None, None, None, FAKE, None, None, None) == C.ERR_BAD_ARG
    assert L.nzb_layernorm_forward(ctypes.byref(d), FAKE + 1, None, None, FAKE, None, None, None) == C.ERR_BAD_ARG
    assert L.nzb_layernorm_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == C.OK and n.value >= 2 * 96 * 4
    assert L.nzb_layernorm_backward(ctypes.byref(_layernorm(ld_dx=95)), FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE,
                                    1 << 30, None) == C.ERR_BAD_ARG
    # nothing is asked for
    assert L.nzb_layernorm_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, None, None, None, None, None, 0, None) == C.OK


def _logprob(**kw):
    d = C.TokenLogprobDesc(rows=5, vocab=300, ld_logits=300, ld_dlogits=300, scale=1.0, dtype=C.F32, index_type=C.I64, top_k=4)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), C.ERR_BAD_ARG), (dict(vocab=-1), C.ERR_BAD_ARG), (dict(ld_logits=299), C.ERR_BAD_ARG),
    (dict(scale=0.0), C.ERR_BAD_ARG), (dict(scale=-1.0), C.ERR_BAD_ARG), (dict(scale=float("nan")), C.ERR_BAD_ARG),
    (dict(scale=float("inf")), C.ERR_BAD_ARG), (dict(scale=9e-5), C.ERR_BAD_ARG), (dict(dtype=3), C.ERR_BAD_ARG), (dict(index_type=-1), C.ERR_BAD_ARG),
    (dict(top_k=33), C.ERR_BAD_ARG), (dict(top_k=-1), C.ERR_BAD_ARG), (dict(vocab=3, top_k=4), C.ERR_BAD_ARG),
    (dict(vocab=0, top_k=0), C.ERR_UNSUPPORTED), (dict(vocab=1 << 29, ld_logits=1 << 29), C.ERR_UNSUPPORTED),
])
def test_token_logprob_refusals(change, code):
    L = C.lib()
    d = _logprob(**change)
    assert L.nzb_token_logprob_forward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == code


def test_token_logprob_pointers():
    L = C.lib()
    d = _logprob()
    assert L.nzb_token_logprob_forward(ctypes.byref(d), None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_forward(ctypes.byref(d), FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_forward(ctypes.byref(d), FAKE + 2, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_forward(ctypes.byref(d), FAKE, FAKE + 4, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_backward(ctypes.byref(d), FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_backward(ctypes.byref(d), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    assert L.nzb_token_logprob_backward(ctypes.byref(_logprob(ld_dlogits=299)), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    d.rows = 0
    assert L.nzb_token_logprob_forward(ctypes.byref(d), None, None, None, None, None, None, None, None) == C.OK


def _ortho(**kw):
    d = C.OrthogonalizeDesc(batch=1, rows=30, cols=40, ld_g=40, stride_g=1200, ld_out=40, stride_out=1200,
                            coef=(ctypes.c_float * 3)(3.4445, -4.775, 2.0315), eps=1e-7, steps=5, dtype=C.F32, out_dtype=C.F32)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), C.ERR_BAD_ARG), (dict(rows=-1), C.ERR_BAD_ARG), (dict(steps=0), C.ERR_BAD_ARG), (dict(steps=65), C.ERR_BAD_ARG),
    (dict(eps=-1.0), C.ERR_BAD_ARG), (dict(ld_g=39), C.ERR_BAD_ARG), (dict(ld_out=39), C.ERR_BAD_ARG), (dict(dtype=5), C.ERR_BAD_ARG),
    (dict(out_dtype=5), C.ERR_BAD_ARG), (dict(batch=70000), C.ERR_UNSUPPORTED), (dict(rows=1 << 25), C.ERR_UNSUPPORTED),
    (dict(rows=1 << 21, cols=1 << 21, ld_g=1 << 21, ld_out=1 << 21), C.ERR_UNSUPPORTED),
])
def test_orthogonalize_refusals(change, code):
    L = C.lib()
    d = _ortho(**change)
    assert L.nzb_orthogonalize(ctypes.byref(d), FAKE, FAKE, FAKE, 1 << 50, None) == code


def test_orthogonalize_workspace():
    L = C.lib()
    d, n, m = _ortho(), ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert L.nzb_orthogonalize_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == C.OK
    assert L.nzb_muon_workspace_bytes(ctypes.byref(d), ctypes.byref(m)) == C.OK and m.value == n.value
    # the fp32 state, two fp16 copies of it, two fp16 squares of the short side
    assert n.value >= 30 * 64 * (4 + 2 * 2) + 2 * 30 * 64 * 2
    assert L.nzb_orthogonalize(ctypes.byref(d), FAKE, FAKE, FAKE, n.value - 1, None) == C.ERR_WORKSPACE
    assert L.nzb_orthogonalize(ctypes.byref(d), FAKE, FAKE, FAKE + 64, n.value, None) == C.ERR_WORKSPACE
    assert L.nzb_orthogonalize(ctypes.byref(d), None, FAKE, FAKE, n.value, None) == C.ERR_BAD_ARG
    assert L.nzb_muon(ctypes.byref(d), FAKE, None, FAKE, .1, 1., .9, 0., 1, FAKE, n.value, None) == C.ERR_BAD_ARG
    d.batch = 0
    assert L.nzb_orthogonalize(ctypes.byref(d), None, None, None, 0, None) == C.OK


def test_descriptor_layouts():
    assert ctypes.sizeof(C.EmbeddingDesc) == 6 * 8 + 6 * 4
    assert ctypes.sizeof(C.LayernormDesc) == 5 * 8 + 4 * 4
    assert ctypes.sizeof(C.TokenLogprobDesc) == 4 * 8 + 4 * 4
    assert ctypes.sizeof(C.OrthogonalizeDesc) == 7 * 8 + 8 * 4


def test_wrappers_refuse_host_tensors_and_bad_shapes():
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: nz.embedding(x, t), lambda: nz.embedding_backward(x, t, x), lambda: nz.layernorm_forward(x),
                 lambda: nz.layernorm_backward(x, x, t, t), lambda: nz.token_logprobs(x, t),
                 lambda: nz.token_logprobs_backward(x, t, t), lambda: nz.orthogonalize(x), lambda: nz.muon_step(x, x, x, 0.1)):
        with pytest.raises(ValueError):
            call()
    from neuzephyr_b200 import ops
    with pytest.raises(ValueError):
        ops._row_stride(torch.zeros(8, 4).t(), "x")
    with pytest.raises(ValueError):
        ops._row_stride(torch.zeros(1, 4).expand(3, 4), "x")
    assert ops._row_stride(torch.zeros(3, 10)[:, :4], "x") == 10
    assert ops._row_stride(torch.zeros(1, 4).expand(1, 4), "x") == 4
    with pytest.raises(ValueError):
        ops._batch_strides(torch.zeros(1, 3, 4).expand(2, 3, 4), "g")
    with pytest.raises(ValueError):
        ops._dtype(t, "x")
    with pytest.raises(ValueError):
        ops._index_type(x, "index")


def test_results_in_place_need_the_same_rows():
    L = C.lib()
    d = _layernorm(ld_y=104)
    assert L.nzb_layernorm_forward(ctypes.byref(d), FAKE, None, None, FAKE, None, None, None) == C.ERR_BAD_ARG
    far = FAKE + (1 << 20)
    d = _layernorm(ld_dx=104)
    for dy, x, dx in ((FAKE, far, FAKE), (far, FAKE, FAKE)):
        assert L.nzb_layernorm_backward(ctypes.byref(d), dy, x, FAKE, FAKE, None, dx, None, None, None, 0, None) == C.ERR_BAD_ARG
    d = _logprob(ld_dlogits=304)
    assert L.nzb_token_logprob_backward(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == C.ERR_BAD_ARG
    d = _ortho(batch=2, stride_out=39)
    assert L.nzb_orthogonalize(ctypes.byref(d), FAKE, FAKE, FAKE, 1 << 30, None) == C.ERR_BAD_ARG
    for w, m, g in ((FAKE, FAKE, far), (far, FAKE, FAKE)):
        assert L.nzb_muon(ctypes.byref(_ortho()), w, m, g, 0.1, 1.0, 0.9, 0.0, 0, FAKE, 1 << 30, None) == C.ERR_BAD_ARG


def test_long_rows_need_a_small_workspace():
    L = C.lib()
    n = ctypes.c_size_t()
    dim = 1 << 20
    d = _layernorm(rows=1000, dim=dim, ld_x=dim, ld_y=dim, ld_dx=dim)
    assert L.nzb_layernorm_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == C.OK and n.value == 64 * 2 * dim * 4


def test_layernorm_results_that_overlap():
    L = C.lib()
    d = _layernorm(overwrite_dx=1, overwrite_dparams=1)
    far = FAKE + (1 << 20)
    for other in (FAKE, FAKE + 4 * 95, FAKE - 4 * 95):  # 96 floats each
        assert L.nzb_layernorm_backward(ctypes.byref(d), far, far, far, far, None, far, FAKE, other, far, 1 << 30, None) == C.ERR_BAD_ARG
        assert b"overlap" in L.nzb_last_error_string()
    for other in (FAKE, FAKE + 4 * 6, FAKE - 4 * 6):  # 7 rows
        assert L.nzb_layernorm_forward(ctypes.byref(d), far, None, None, far, FAKE, other, None) == C.ERR_BAD_ARG
        assert b"overlap" in L.nzb_last_error_string()
