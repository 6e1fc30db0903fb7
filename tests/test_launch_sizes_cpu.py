"""Calls whose launch would have 2^32 threads or more are refused by the entry,
before the launch.  (No GPU is asked: nothing is launched, no pointer read.)"""

import ctypes

import pytest
import torch

from refinekv import _hip

INVALID = 1
AT = 1 << 44  # (addresses that no array of these calls comes near)


def places(kind, **fields):
    """A cache of 2^20 sequences of a page each, 1 head of 32 dims."""
    return kind(block_table=AT, table_stride=1, lengths=AT + (1 << 30), pages=4, heads=1,
                page_size=16, dim=32, sequences=1 << 20, max_blocks=1,
                dtype=_hip.DTYPE_CODES[torch.bfloat16], **fields)


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def refused(lib, rc):
    assert rc == INVALID, (rc, lib.rkv_last_error())
    assert b"too many tokens" in lib.rkv_last_error()


def paged():
    strides = (ctypes.c_int64 * 3)(512, 512, 32)
    return places(_hip._PagedCache, keys=2 * AT, values=3 * AT, key_strides=strides,
                  value_strides=strides)


def quantized():
    return places(_hip._QuantizedCache, key_codes=2 * AT, value_codes=3 * AT, key_scales=4 * AT,
                  value_scales=5 * AT)


# a row of 32 dims takes 4 threads of a vector of 8 dims, keys and values 8
FEW = 1 << 29  # tokens: 2^32 threads of the reads


@pytest.mark.parametrize("tokens", [FEW, FEW + 12345, 1 << 34, (1 << 37) - 1])
def test_reads(lib, tokens):
    refused(lib, lib.rkv_paged_read(ctypes.byref(paged()), tokens, AT, 8 * AT, 16 * AT, 0))
    refused(lib, lib.rkv_quantized_read(ctypes.byref(quantized()), tokens, AT, 8 * AT, 16 * AT, 0))


@pytest.mark.parametrize("tokens", [FEW, 1 << 34])
def test_appends(lib, tokens):
    rows = [v for at in (8 * AT, 16 * AT) for v in (at, 32, 32)]
    none = (0, 0, 0, 0, 0, 0, 0)
    refused(lib, lib.rkv_quantized_append(ctypes.byref(quantized()), *none, *rows, tokens, AT, 0, 0,
                                          0, 1.0, 0))
    refused(lib, lib.rkv_paged_append(ctypes.byref(paged()), *none, *rows, 2 * tokens, AT, 0, 0, 0,
                                      1.0, 0))


def test_rotary(lib):
    tokens = 1 << 35
    refused(lib, lib.rkv_rotary(8 * AT, 32, 32, 1, 0, 0, 0, 0, 1, tokens, 32, 2 * AT, 0, 3 * AT, 32,
                                0, 1.0, 0, 8 * AT, 32, 32, 0, 0, 0, 0))
