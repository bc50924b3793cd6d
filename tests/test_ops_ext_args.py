"""Refusals of the sampling, top-k, distillation and shared-prefix attention
entry points. Every case returns CNGPT_ERR_ARG before anything is launched, so
they run without a GPU."""
import ctypes as C

import numpy as np
import pytest

from cngpt_b200 import abi

HOST = np.zeros(64, np.float32)
P = HOST.ctypes.data


def refused(lib, status, text):
    assert status == abi.ERR_ARG
    assert text in lib.cngpt_cuda_last_message().decode(), lib.cngpt_cuda_last_message()
    lib.cngpt_cuda_clear_status()


@pytest.mark.parametrize("ld,rows,vocab,text", [(8, -1, 8, "bad shape"), (8, 1, 0, "bad shape"), (7, 1, 8, "bad shape"),
                                                (300000, 1, 262145, "unsupported")])
def test_sample_refuses_bad_shapes(lib, ld, rows, vocab, text):
    refused(lib, lib.cngpt_cuda_sample(P, ld, rows, vocab, None, None, None, None, P, P, None), text)


@pytest.mark.parametrize("k", [0, -1, 9, 1025])
def test_topk_refuses_bad_k(lib, k):
    refused(lib, lib.cngpt_cuda_topk(P, 8 if k < 10 else 5000, 1, 8 if k < 10 else 5000, k, P, P), "k=")


@pytest.mark.parametrize("tau,alpha", [(0.0, 1.0), (-1.0, 1.0), (float("nan"), 1.0), (float("inf"), 1.0), (1.0, -0.1),
                                       (1.0, 1.1), (1.0, float("nan"))])
def test_distill_refuses_bad_parameters(lib, tau, alpha):
    refused(lib, lib.cngpt_cuda_distill(P, 8, 1, 8, P, P, 2, P, tau, alpha, 1.0, P, P, None, 0), "temperature")


@pytest.mark.parametrize("k", [-1, 1025])
def test_distill_refuses_bad_k(lib, k):
    refused(lib, lib.cngpt_cuda_distill(P, 8, 1, 8, P, P, k, P, 1.0, 1.0, 1.0, P, P, None, 0), "k=")


def test_host_and_null_and_misaligned_pointers_are_refused(lib):
    refused(lib, lib.cngpt_cuda_sample(P, 8, 1, 8, None, None, None, None, P, P, None), "device pointer")
    refused(lib, lib.cngpt_cuda_sample(None, 8, 1, 8, None, None, None, None, P, P, None), "NULL")
    refused(lib, lib.cngpt_cuda_sample(P + 2, 8, 1, 8, None, None, None, None, P, P, None), "aligned")
    refused(lib, lib.cngpt_cuda_topk(P, 8, 1, 8, 2, P, P), "device pointer")
    refused(lib, lib.cngpt_cuda_distill(P, 8, 1, 8, P, P, 2, P, 1.0, 1.0, 1.0, P, P, None, 0), "device pointer")
    refused(lib, lib.cngpt_cuda_prefix_attention(P, 8, P, P, 8, 1, P, P, 8, 8, P, 1, P, 8, 1, 1, 1, 8, 1.0, P, 1 << 20),
            "device pointer")


def test_rows_of_zero_are_nothing_to_do(lib):
    assert lib.cngpt_cuda_sample(None, 8, 0, 8, None, None, None, None, None, None, None) == abi.OK
    assert lib.cngpt_cuda_topk(None, 8, 0, 8, 2, None, None) == abi.OK
    assert lib.cngpt_cuda_prefix_attention(None, 8, None, None, 8, 0, None, None, 8, 8, None, 0, None, 8, 0, 1, 1, 8, 1.0,
                                           None, 0) == abi.OK


@pytest.mark.parametrize("B,H,Hk,hs,Pn,S", [(-1, 1, 1, 8, 1, 1), (1, 0, 1, 8, 1, 1), (1, 4, 3, 8, 1, 1), (1, 4, 0, 8, 1, 1),
                                            (1, 4, 4, 0, 1, 1), (1, 4, 4, 257, 1, 1), (1, 4, 4, 8, -1, 1),
                                            (1, 4, 4, 8, 1, -1)])
def test_prefix_attention_refuses_bad_shapes(lib, B, H, Hk, hs, Pn, S):
    refused(lib, lib.cngpt_cuda_prefix_attention(P, 1 << 12, P, P, 1 << 12, Pn, P, P, 1 << 12, 1 << 20, P, S, P, 1 << 12, B, H,
                                                 Hk, hs, 1.0, P, 1 << 20), "bad shape")
    assert lib.cngpt_cuda_prefix_attention_workspace(B, H, Hk, hs, Pn, S) == 0
    lib.cngpt_cuda_clear_status()


@pytest.mark.parametrize("ldq,ldp,lds,stride,ldo", [(31, 32, 32, 160, 32), (32, 31, 32, 160, 32), (32, 32, 31, 160, 32),
                                                    (32, 32, 32, 159, 32), (32, 32, 32, 160, 31)])
def test_prefix_attention_refuses_bad_pitches(lib, ldq, ldp, lds, stride, ldo):
    refused(lib, lib.cngpt_cuda_prefix_attention(P, ldq, P, P, ldp, 3, P, P, lds, stride, P, 5, P, ldo, 2, 4, 4, 8, 1.0, P,
                                                 1 << 20), "bad pitch")
