"""Training-side operators on a host without a GPU: argument checks of the C ABI
(all made before a device is touched), no CPU fallback, module construction."""
import ctypes

import pytest
import torch

import grad_clip
import group_norm_act as gna
import scaled_embedding as emb
from bevk import cabi


def _gn(**kw):
    p = cabi.GroupNormProblem()
    p.dtype, p.param_dtype = cabi.DTYPE_F16, cabi.DTYPE_F32
    p.batch, p.channels, p.groups, p.pixels = 2, 64, 8, 100
    p.act, p.eps = cabi.ACT_SILU, 1e-5
    for name in ("input_strides", "output_strides", "grad_output_strides"):
        getattr(p, name)[0], getattr(p, name)[1] = 6400, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status,word", [
    (dict(groups=7), cabi.ERR_INVALID_ARGUMENT, "divide"),
    (dict(groups=0), cabi.ERR_INVALID_ARGUMENT, "sizes"),
    (dict(channels=0), cabi.ERR_INVALID_ARGUMENT, "sizes"),
    (dict(batch=-1), cabi.ERR_INVALID_ARGUMENT, "sizes"),
    (dict(dtype=cabi.DTYPE_F64), cabi.ERR_UNSUPPORTED, "dtype"),
    (dict(param_dtype=cabi.DTYPE_BF16), cabi.ERR_UNSUPPORTED, "parameter dtype"),
    (dict(act=7), cabi.ERR_UNSUPPORTED, "activation"),
    (dict(eps=float("nan")), cabi.ERR_INVALID_ARGUMENT, "eps"),
    (dict(eps=-1.0), cabi.ERR_INVALID_ARGUMENT, "eps"),
    (dict(pixels=1 << 31), cabi.ERR_INDEX_OVERFLOW, "pixels"),
])
def test_group_norm_problem_validation(kw, status, word):
    L, p = cabi.lib(), _gn(**kw)
    assert L.bevk_group_norm_act_workspace_bytes(ctypes.byref(p), 0) == 0
    st = L.bevk_group_norm_act_forward(ctypes.byref(p), 16, None, None, 16, None, None, 16, 1 << 20,
                                       None)
    assert st == status and word in cabi.last_error()
    st = L.bevk_group_norm_act_backward(ctypes.byref(p), 16, 16, 16, 16, None, None, 16, None, None,
                                        16, 1 << 20, None)
    assert st == status


def test_group_norm_pointer_checks():
    L, p = cabi.lib(), _gn()
    assert L.bevk_group_norm_act_workspace_bytes(ctypes.byref(p), 0) > 0
    assert L.bevk_group_norm_act_workspace_bytes(ctypes.byref(p), 1) > 0
    ref = ctypes.byref(p)
    assert L.bevk_group_norm_act_forward(ref, None, None, None, 16, None, None, 16, 1 << 20,
                                         None) == cabi.ERR_INVALID_ARGUMENT
    assert L.bevk_group_norm_act_forward(ref, 16, None, None, 16, 16, None, 16, 1 << 20,
                                         None) == cabi.ERR_INVALID_ARGUMENT
    assert L.bevk_group_norm_act_forward(ref, 16, None, None, 16, None, None, 8, 1 << 20,
                                         None) == cabi.ERR_MISALIGNED
    assert L.bevk_group_norm_act_forward(None, 16, None, None, 16, None, None, 16, 1 << 20,
                                         None) == cabi.ERR_INVALID_ARGUMENT
    # nothing to do
    empty = _gn(batch=0)
    assert L.bevk_group_norm_act_forward(ctypes.byref(empty), None, None, None, None, None, None,
                                         None, 0, None) == cabi.OK
    assert L.bevk_group_norm_act_backward(ref, 16, 16, 16, 16, None, None, None, None, None, None,
                                          0, None) == cabi.OK


def test_group_norm_module_and_no_cpu_fallback():
    m = gna.GroupNormAct(8, 32, act="relu")
    assert set(m.state_dict()) == {"weight", "bias"} and "relu" in repr(m)
    assert not gna.GroupNormAct(8, 32, affine=False).state_dict()
    with pytest.raises(ValueError):
        gna.GroupNormAct(5, 32)
    with pytest.raises(ValueError, match="act"):
        gna.GroupNormAct(8, 32, act="tanh")
    with pytest.raises(RuntimeError, match="CUDA"):
        m(torch.randn(1, 32, 2, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        gna.group_norm_act_backward(*[torch.randn(1, 32, 2, 2)] * 2, torch.ones(1, 8),
                                    torch.ones(1, 8), 8)


def test_grad_clip_checks():
    L = cabi.lib()
    assert L.bevk_grad_clip_workspace_bytes(0) > 0
    assert L.bevk_grad_clip_workspace_bytes(2300) > L.bevk_grad_clip_workspace_bytes(1000)
    t = (cabi.GradTensor * 2)()
    for k in range(2):
        t[k].grad, t[k].out, t[k].numel = 4096, 4096, 8

    def call(n=2, kind=0, limit=1.0, scale=1, norm=16, ws=16, nbytes=1 << 20):
        return L.bevk_grad_clip(t, n, kind, limit, 1e-6, scale, norm, ws, nbytes, None)

    assert call() == cabi.ERR_INVALID_ARGUMENT and "overlaps" in cabi.last_error()
    t[1].grad = t[1].out = 4096 + 32
    assert call(kind=2) == cabi.ERR_UNSUPPORTED
    assert call(limit=-1.0) == cabi.ERR_INVALID_ARGUMENT
    assert call(limit=float("nan")) == cabi.ERR_INVALID_ARGUMENT
    assert call(norm=None) == cabi.ERR_INVALID_ARGUMENT
    assert call(n=-1) == cabi.ERR_INVALID_ARGUMENT
    assert call(nbytes=8) == cabi.ERR_WORKSPACE
    assert call(ws=None) == cabi.ERR_WORKSPACE
    assert call(ws=24) == cabi.ERR_MISALIGNED
    t[1].out = 4096 + 24                     # overlaps the first tensor, which is written
    assert call() == cabi.ERR_INVALID_ARGUMENT
    t[1].out = t[1].grad
    t[1].grad_dtype, t[1].out_dtype = cabi.DTYPE_F16, cabi.DTYPE_F32
    assert call() == cabi.ERR_INVALID_ARGUMENT and "two types" in cabi.last_error()
    t[1].grad_dtype = cabi.DTYPE_F64
    assert call() == cabi.ERR_UNSUPPORTED
    t[1].numel = -1
    assert call() == cabi.ERR_INVALID_ARGUMENT
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_clip.grad_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="norm_type"):
        grad_clip.clip_grads([torch.ones(3)], 1.0, norm_type=3)
    with pytest.raises(TypeError):
        grad_clip.clip_grad_norm_(3.0, 1.0)
    assert float(grad_clip.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0


def test_embedding_checks():
    L = cabi.lib()
    a = cabi.EmbeddingBackwardArgs()

    def reset(**kw):
        a.num_ids, a.num_rows, a.dim, a.ids_are_64bit = 10, 20, 8, 1
        a.grad_output_ld = a.grad_table_ld = 8
        a.padding_idx, a.scale, a.accumulate = -1, 1.0, 0
        a.grad_output_dtype = a.grad_table_dtype = cabi.DTYPE_BF16
        for k, v in kw.items():
            setattr(a, k, v)

    def call(dy=16, ids=16, out=16, ws=256, nbytes=1 << 30):
        return L.bevk_embedding_backward(ctypes.byref(a), dy, ids, out, ws, nbytes, None)

    for kw, status in ((dict(grad_output_dtype=cabi.DTYPE_F64), cabi.ERR_UNSUPPORTED),
                       (dict(grad_table_dtype=cabi.DTYPE_F16), cabi.ERR_UNSUPPORTED),
                       (dict(num_ids=-1), cabi.ERR_INVALID_ARGUMENT),
                       (dict(dim=0), cabi.ERR_INVALID_ARGUMENT),
                       (dict(grad_table_ld=7), cabi.ERR_INVALID_ARGUMENT),
                       (dict(num_ids=1 << 31), cabi.ERR_INDEX_OVERFLOW),
                       (dict(num_rows=1 << 31), cabi.ERR_INDEX_OVERFLOW)):
        reset(**kw)
        assert L.bevk_embedding_backward_workspace_bytes(ctypes.byref(a)) == 0
        assert call() == status, kw
    reset()
    assert L.bevk_embedding_backward_workspace_bytes(ctypes.byref(a)) > 0
    assert call(dy=None) == cabi.ERR_INVALID_ARGUMENT
    assert call(out=None) == cabi.ERR_INVALID_ARGUMENT
    assert call(nbytes=64) == cabi.ERR_WORKSPACE
    assert call(ws=128) == cabi.ERR_MISALIGNED
    reset(num_rows=0)
    assert call(out=None) == cabi.OK
    reset(num_ids=0, accumulate=1)
    assert call(dy=None, ids=None, ws=None, nbytes=0) == cabi.OK

    def look(ld=8, n=4, rows=20, dim=8, dtype=cabi.DTYPE_F32, ids=16):
        return L.bevk_embedding_forward(16, ld, ids, 1, n, rows, dim, 1.0, 16, dtype, None)

    assert look(dtype=cabi.DTYPE_F64) == cabi.ERR_UNSUPPORTED
    assert look(n=-1) == cabi.ERR_INVALID_ARGUMENT and look(dim=0) == cabi.ERR_INVALID_ARGUMENT
    assert look(ids=None) == cabi.ERR_INVALID_ARGUMENT
    assert look(n=0) == cabi.OK


def test_embedding_module_and_no_cpu_fallback():
    m = emb.ScaledEmbedding(10, 4, padding_idx=-1, scale=2.0)
    assert set(m.state_dict()) == {"weight"} and not m.weight[9].any() and "scale=2.0" in repr(m)
    with pytest.raises(ValueError, match="padding_idx"):
        emb.ScaledEmbedding(10, 4, padding_idx=10)
    with pytest.raises(RuntimeError, match="CUDA"):
        m(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        emb.scaled_embedding_backward(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64), 10)
