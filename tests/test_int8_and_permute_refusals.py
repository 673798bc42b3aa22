"""Calls that w8a8_int8_matmul, w8a8_int8_grouped_mm, per_token_quant_int8, moe_permute and moe_unpermute refuse (no GPU)."""
import pytest
import torch
from torch.autograd import forward_ad

import flag_gems
from flaggems_b200 import _cabi

I8 = torch.int8


def _mm(**over):
    args = dict(A=torch.zeros(3, 32, dtype=I8), B=torch.zeros(5, 32, dtype=I8), As=torch.ones(3, 1), Bs=torch.ones(5))
    return flag_gems.w8a8_int8_matmul(**{**args, **over})


def _grouped(**over):
    args = dict(A=torch.zeros(3, 32, dtype=I8), B=torch.zeros(2, 5, 32, dtype=I8), As=torch.ones(3), Bs=torch.ones(2, 5),
                offs=torch.tensor([1, 3], dtype=torch.int32))
    return flag_gems.w8a8_int8_grouped_mm(**{**args, **over})


def _permute(**over):
    args = dict(hidden_states=torch.zeros(3, 16), topk_ids=torch.zeros(3, 2, dtype=torch.int32), num_experts=4)
    return flag_gems.moe_permute(**{**args, **over})


def _unpermute(**over):
    ids = torch.zeros(3, 2, dtype=torch.int32)
    args = dict(rows=torch.zeros(6, 16), plan=flag_gems.MoEPermutation(ids[0], ids, ids.view(-1)), topk_weights=torch.ones(3, 2))
    return flag_gems.moe_unpermute(**{**args, **over})


def test_ordinary_calls_want_a_gpu():
    for call in (_mm, _grouped, _permute, _unpermute, lambda: flag_gems.per_token_quant_int8(torch.zeros(2, 16))):
        with pytest.raises(_cabi.FlagGemsB200Error, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("over,error,text", [
    (dict(A=torch.zeros(3, 48, dtype=I8)), AssertionError, "48 values per row"),
    (dict(B=torch.zeros(5, dtype=I8)), AssertionError, r"B \[N, K\]"),
    (dict(A=torch.zeros(3, 32)), NotImplementedError, "must be int8"),
    (dict(B=torch.zeros(5, 32, dtype=torch.uint8)), NotImplementedError, "must be int8"),
    (dict(A=torch.zeros(3, 24, dtype=I8), B=torch.zeros(5, 24, dtype=I8)), NotImplementedError, "multiple of 16"),
    (dict(A=torch.zeros(3, 0, dtype=I8), B=torch.zeros(5, 0, dtype=I8)), NotImplementedError, "positive multiple of 16"),
    (dict(A=torch.zeros(3, 131072, dtype=I8), B=torch.zeros(5, 131072, dtype=I8)), NotImplementedError, "at most 131071"),
    (dict(output_dtype=torch.int32), NotImplementedError, "output dtype"),
    (dict(As=torch.ones(5, 1)), AssertionError, "As must be"),
    (dict(As=torch.ones(1, 3)), AssertionError, "As must be"),
    (dict(Bs=torch.ones(1, 5)), AssertionError, "Bs must be"),
    (dict(bias=torch.ones(1, 5)), AssertionError, "bias must have shape"),
    (dict(bias=torch.ones(5, dtype=torch.float64)), NotImplementedError, "bias dtype"),
])
def test_matmul(over, error, text):
    with pytest.raises(error, match=text):
        _mm(**over)


@pytest.mark.parametrize("over,error,text", [
    (dict(B=torch.zeros(5, 32, dtype=I8)), AssertionError, r"B \[G, N, K\]"),
    (dict(A=torch.zeros(3, 16, dtype=I8)), AssertionError, "16 values per row"),
    (dict(A=torch.zeros(3, 32, dtype=torch.float8_e4m3fn)), NotImplementedError, "must be int8"),
    (dict(As=torch.ones(1)), AssertionError, "As must have shape"),
    (dict(Bs=torch.ones(5)), AssertionError, "Bs must have shape"),
    (dict(offs=torch.tensor([3], dtype=torch.int32)), AssertionError, "offs must be int32"),
    (dict(offs=torch.tensor([1, 3])), AssertionError, "offs must be int32"),
    (dict(bias=torch.ones(3, 5)), AssertionError, "bias must have shape"),
    (dict(output_dtype=I8), NotImplementedError, "output dtype"),
])
def test_grouped(over, error, text):
    with pytest.raises(error, match=text):
        _grouped(**over)


def _quant(x):
    return flag_gems.per_token_quant_int8(x)


GRADIENTS = [(_mm, "As", (3, 1)), (_mm, "Bs", (5,)), (_mm, "bias", (5,)), (_grouped, "As", (3,)), (_grouped, "Bs", (2, 5)),
             (_grouped, "bias", (2, 5)), (_quant, "x", (2, 16))]


@pytest.mark.parametrize("call,name,shape", GRADIENTS)
def test_gradients_that_would_be_lost(call, name, shape):
    t = torch.ones(shape, requires_grad=True)
    with pytest.raises(NotImplementedError, match=f"{name} has no gradient"):
        call(**{name: t})
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t.detach(), torch.ones(shape))
        with pytest.raises(NotImplementedError, match=f"{name} has no gradient"), torch.no_grad():
            call(**{name: dual})
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(_cabi.FlagGemsB200Error, match="CUDA tensors only"):
            call(**{name: dual})
    with torch.no_grad(), pytest.raises(_cabi.FlagGemsB200Error, match="CUDA tensors only"):
        call(**{name: t})


@pytest.mark.parametrize("over,error,text", [
    (dict(topk_ids=torch.zeros(3, dtype=torch.int32)), AssertionError, "topk_ids must be"),
    (dict(topk_ids=torch.zeros(3, 2)), NotImplementedError, "int32 or int64"),
    (dict(topk_ids=torch.zeros(2, 2, dtype=torch.int32)), AssertionError, "3 tokens, 2 rows"),
    (dict(hidden_states=torch.zeros(3, 2, 8)), AssertionError, "hidden_states must be 2-D"),
    (dict(hidden_states=torch.zeros(3, 16, dtype=torch.float64)), NotImplementedError, "unsupported dtype"),
    (dict(num_experts=0), AssertionError, "num_experts must be positive"),
    (dict(scale=torch.ones(3, 1, dtype=torch.float16)), AssertionError, "scale must be float32"),
    (dict(scale=torch.ones(3)), AssertionError, "scale must be 2-D"),
    (dict(scale=torch.ones(2, 1)), AssertionError, "2 rows of scales"),
    (dict(scale=torch.ones(3, 1, requires_grad=True)), NotImplementedError, "scale has no gradient"),
])
def test_permute(over, error, text):
    with pytest.raises(error, match=text):
        _permute(**over)


@pytest.mark.parametrize("over,error,text", [
    (dict(rows=torch.zeros(5, 16)), AssertionError, "the plan has 6 rows, got 5"),
    (dict(rows=torch.zeros(6, 16, dtype=I8)), NotImplementedError, "unsupported dtype"),
    (dict(rows=torch.zeros(6)), AssertionError, "rows must be 2-D"),
    (dict(topk_weights=torch.ones(6)), AssertionError, "topk_weights must have shape"),
    (dict(topk_weights=torch.ones(3, 2, dtype=torch.float64)), NotImplementedError, "topk_weights"),
    (dict(plan=flag_gems.MoEPermutation(None, torch.zeros(3, 2), None)), AssertionError, "row_of_slot must be int32"),
])
def test_unpermute(over, error, text):
    with pytest.raises(error, match=text):
        _unpermute(**over)


@pytest.mark.skipif(torch.cuda.is_available(), reason="passes made-up addresses: for hosts where nothing can be launched")
def test_entry_points_check_their_sizes():
    lib, p = _cabi.lib(), 4096

    def refused(rc, code, text):
        assert rc == code and text in lib.fg_last_error().decode(), (rc, lib.fg_last_error())

    def mm(m=4, n=4, k=16, lda=16, out=0, bias=0, a=p):
        return lib.fg_scaled_mm_int8(p, a, p, p, p, p, bias, m, n, k, lda, k, n, 1, 1, out, 0, None)

    refused(mm(k=131072, lda=131072), -2, "may leave 32 bits")
    refused(mm(k=24, lda=32), -2, "multiple of 16")
    refused(mm(lda=0), -1, "row stride smaller")
    refused(mm(a=p + 8), -2, "16-byte aligned")
    refused(mm(out=3), -1, "bad out_dtype")
    refused(mm(bias=7), -1, "bad bias_dtype")
    refused(mm(m=-1), -1, "negative size")
    refused(lib.fg_scaled_mm_int8(p, None, p, p, p, None, 0, 4, 4, 16, 16, 16, 4, 1, 1, 0, 0, None), -1, "null pointer")
    assert mm(m=0) == 0 and mm(n=0) == 0
    need = lib.fg_scaled_grouped_mm_workspace_bytes(100, 2, 128)
    refused(lib.fg_scaled_grouped_mm_int8(p, p, p, p, p, None, 0, p, 2, 100, 64, 128, 128, 64, 0, p, need - 1, None), -1, "workspace holds")
    refused(lib.fg_scaled_grouped_mm_int8(p, p, p, p, p, None, 0, p, 1025, 100, 64, 128, 128, 64, 0, p, need, None), -2, "1024 groups")
    refused(lib.fg_scaled_grouped_mm_int8(p, p, p, p, p, None, 0, p, 2, 100, 64, 131072, 131072, 64, 0, p, need, None), -2, "32 bits")

    def permute(t=4, topk=2, e=4, h=8, esz=2, offs=p, rows=p, cols=0, map_=None, map_len=0, ws=0):
        return lib.fg_moe_permute(rows, None, offs, p, p, p, None, p, 0, map_, map_len, t, topk, e, h, esz, h, cols, cols, p, ws, None)

    refused(permute(e=1025), -2, "num_experts 1025")
    refused(permute(e=0), -2, "num_experts 0")
    refused(permute(t=1 << 30), -2, "size too large")
    refused(permute(esz=3), -1, "elements of 3 bytes")
    refused(permute(t=-1), -1, "negative size")
    refused(permute(offs=None), -1, "null pointer")
    refused(permute(rows=None), -1, "null pointer")
    refused(permute(cols=2), -1, "null pointer")
    refused(permute(map_=p), -1, "empty expert_map")
    for t, topk, e in ((10000, 8, 256), (1 << 20, 8, 1024), (4097, 1, 1), (1 << 27, 15, 3)):
        need = lib.fg_moe_permute_workspace_bytes(t, topk, e)
        assert 0 < need <= 256 * (e + 1) * 8
        refused(permute(t=t, topk=topk, e=e, ws=need - 1), -1, "workspace holds")
    assert lib.fg_moe_permute_workspace_bytes(64, 8, 1024) == 0 and lib.fg_moe_permute_workspace_bytes(1 << 30, 2, 8) == -1
    refused(lib.fg_moe_unpermute(p, p, p, p, 3, 4, 2, 8, 8, 8, 2, 0, None), -1, "bad weight dtype")
    refused(lib.fg_moe_unpermute(p, p, p, None, 0, 4, 2, 8, 8, 8, 2, 3, None), -1, "unsupported dtype")
    refused(lib.fg_moe_unpermute(p, p, None, None, 0, 4, 2, 8, 8, 8, 2, 0, None), -1, "null pointer")
    assert lib.fg_moe_unpermute(p, p, p, None, 0, 0, 2, 0, 8, 8, 2, 0, None) == 0
    refused(lib.fg_moe_unpermute_backward(p, p, p, p, p, p, 5, 4, 2, 8, 8, 8, 8, 2, 0, None), -1, "bad weight dtype")
    refused(lib.fg_moe_unpermute_backward(p, p, p, None, p, p, 2, 4, 2, 8, 8, 8, 8, 2, 0, None), -1, "null pointer")
    assert lib.fg_moe_unpermute_backward(p, p, p, p, p, p, 2, 0, 2, 8, 8, 8, 8, 2, 0, None) == 0


@pytest.mark.parametrize("expert_map,error,text", [
    (torch.zeros(4), NotImplementedError, "expert_map must be int32 or int64"),
    (torch.zeros(0, dtype=torch.int32), AssertionError, "1-D and not empty"),
    (torch.zeros(2, 2, dtype=torch.int32), AssertionError, "1-D and not empty"),
])
def test_expert_maps(expert_map, error, text):
    with pytest.raises(error, match=text):
        _permute(expert_map=expert_map)


@pytest.mark.parametrize("call,name,shape", [(_permute, "hidden_states", (3, 16)), (_permute, "scale", (3, 1)), (_unpermute, "rows", (6, 16)),
                                             (_unpermute, "topk_weights", (3, 2))])
def test_forward_mode(call, name, shape):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            call(**{name: forward_ad.make_dual(torch.ones(shape), torch.ones(shape))})


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_gradients_of_8_bit_floats(dtype):
    x = torch.zeros(3, 16).to(dtype).requires_grad_()
    with pytest.raises(NotImplementedError, match="have no gradient"):
        _permute(hidden_states=x)
    with torch.no_grad(), pytest.raises(_cabi.FlagGemsB200Error, match="CUDA tensors only"):
        _permute(hidden_states=x)
