"""Refusals of the routing statistics' entry points: nothing here touches a GPU."""
import ctypes as C

import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _capi as capi

FAKE = 0x7f0000000100  # never dereferenced


def counts(temp=FAKE, have=1 << 20, ids=FAKE, rows=10, k=2, stride=2, width=8, experts=8, out=FAKE, begins=FAKE):
    n = C.c_size_t(have)
    return capi.lib.tb200_expert_counts(temp, C.byref(n), ids, rows, k, stride, width, None, experts, out, begins, None)


def balance(temp=FAKE, have=1 << 20, z=FAKE, dtype=capi.BF16, ids=FAKE, k=2, stride=2, width=8, offsets=None, ob=0, seqs=1,
            rows=10, experts=8, out=FAKE):
    n, r = C.c_size_t(have), capi.Rows(z, experts, 0)
    return capi.lib.tb200_balance_loss(temp, C.byref(n), C.byref(r), dtype, ids, k, stride, width, None, offsets, ob, seqs,
                                       rows, experts, out, out, out, None)


def backward(z=FAKE, dtype=capi.F16, weights=FAKE, dloss=FAKE, offsets=None, ob=0, seqs=1, rows=10, experts=8, out=FAKE):
    r, o = capi.Rows(z, experts, 0), capi.Rows(out, experts, 0)
    return capi.lib.tb200_balance_loss_backward(C.byref(r), dtype, weights, dloss, None, offsets, ob, seqs, rows, experts,
                                                C.byref(o), None)


def test_counts_refusals():
    assert counts(temp=None) == 0
    assert counts(experts=0) == counts(k=0) == counts(width=2) == counts(stride=1) == capi.ERR_INVALID_ARGUMENT
    assert counts(ids=None) == counts(ids=FAKE + 4) == counts(out=None) == counts(begins=FAKE + 4) == capi.ERR_INVALID_ARGUMENT
    assert counts(temp=FAKE + 8) == capi.ERR_INVALID_ARGUMENT and counts(have=100) == capi.ERR_TEMP_TOO_SMALL
    assert counts(experts=8193) == capi.ERR_UNSUPPORTED


def test_balance_refusals():
    assert balance(temp=None) == 0
    assert balance(dtype=capi.F64) == balance(experts=1025) == capi.ERR_UNSUPPORTED
    assert balance(experts=0) == balance(seqs=2) == balance(ob=2) == balance(ob=4) == capi.ERR_INVALID_ARGUMENT
    assert balance(z=FAKE + 1) == balance(ids=None) == balance(out=None) == balance(out=FAKE + 4) == capi.ERR_INVALID_ARGUMENT
    assert balance(ob=8, offsets=FAKE + 4) == capi.ERR_INVALID_ARGUMENT and balance(have=100) == capi.ERR_TEMP_TOO_SMALL


def test_backward_refusals():
    assert backward(rows=0) == 0
    assert backward(dtype=capi.I32) == backward(experts=2000) == capi.ERR_UNSUPPORTED
    assert backward(experts=0) == backward(seqs=0) == backward(weights=None) == backward(dloss=FAKE + 2) == capi.ERR_INVALID_ARGUMENT
    assert backward(out=None) == backward(z=FAKE + 1) == backward(ob=4) == capi.ERR_INVALID_ARGUMENT


def test_python_front_end_refuses_cpu_tensors():
    z, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    for call in (lambda: tb.expert_counts(ids, 8), lambda: tb.balance_loss(z, ids), lambda: tb.balance_loss_backward(z, z, z)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_numbers_beyond_32_bits_are_refused():
    """The library takes experts and ids a row in 32 bits: 2^32 + 8 experts must not be taken for 8."""
    ops, wide = tb.model_ops, (1 << 32) + 8
    assert ops._counts_bytes(8) >= 256
    for experts in (wide, -1, 8 - (1 << 32)):
        with pytest.raises(ValueError):
            ops._counts_bytes(experts)
    assert ops._ids(torch.empty(3, 8, dtype=torch.int32, device="meta")) == (3, 8, 8, 4)
    assert ops._logits(torch.empty(3, 8, device="meta"), None)[-1] == 8
    with pytest.raises(ValueError):
        ops._ids(torch.empty(3, wide, dtype=torch.int32, device="meta"))
    with pytest.raises(ValueError):
        ops._logits(torch.empty(3, wide, device="meta"), None)
