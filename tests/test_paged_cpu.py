"""The paged operators' boundary and format without a GPU: the header, its ctypes and Rust tables, refusals that come before any GPU
work, and what the format promises."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import bonsai_pot_b200 as bp
from bonsai_pot_b200 import _lib
from tests import paged_ref as R
from tests.test_ffi_crate import header_functions, rust_functions

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "bonsai_paged.h")
RS = os.path.join(ROOT, "ffi", "bonsai-attn-sys", "src", "paged.rs")
STRUCTS = {"bp_rope_table": _lib.RopeTableStruct, "bp_rope_config": _lib.RopeConfigStruct, "bp_rows": _lib.RowsStruct, "bp_kv4_pool": _lib.PoolStruct,
           "bp_kv4_attn": _lib.AttnStruct}


def text(path):
    return re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)


def test_ctypes_and_rust_tables_cover_the_header():
    h = header_functions(HEADER)
    lib = _lib.load()
    assert sorted(h) == sorted(_lib.PAGED_SIGNATURES) and len(h) == 10
    for name, (n_args, is_void) in h.items():
        assert hasattr(lib, name)
        res, args = _lib.PAGED_SIGNATURES[name]
        assert len(args) == n_args and (res is None) == is_void, name
    assert h == rust_functions(RS)


def test_structs_and_constants_match_the_header():
    rust = re.sub(r"//.*", "", open(RS).read())
    for name, cls in STRUCTS.items():
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text(HEADER), flags=re.S).group(1)
        want = []
        for decl in body.split(";"):
            decl = decl.strip()
            if decl:
                want += [n.strip().lstrip("*") for n in re.sub(r"^(const )?\w+\*? ", "", decl).split(",")]
        assert [f[0] for f in cls._fields_] == want, name
        fields = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, flags=re.S).group(1)
        assert re.findall(r"pub (\w+):", fields) == want, name
    enum = dict(re.findall(r"\b(BP_(?:DTYPE|ROPE)_[A-Z0-9_]+)\s*=\s*(\d+)", text(HEADER)))
    assert enum == dict(re.findall(r"pub const (BP_[A-Z0-9_]+): u32 = (\d+);", rust)) and len(enum) == 8


def test_pool_sizes():
    assert bp.KV4Pool.bytes(3, 16, 2, 128) == 3 * 16 * 2 * 160
    assert bp.KV4Pool.bytes(1 << 20, 64, 8, 64) == (1 << 20) * 64 * 8 * 80  # beyond 32 bits
    for bad in ((0, 16, 1, 64), (1, 48, 1, 64), (1, 16, 0, 64), (1, 16, 1, 96), (-1, 16, 1, 64), (1, 128, 1, 64)):
        with pytest.raises(bp.ConfigError):
            bp.KV4Pool.bytes(*bad)


def test_nothing_runs_without_a_context_or_a_device():
    lib = _lib.load()
    assert lib.bp_paged_create(0, None) == 7
    assert lib.bp_paged_status(None, None) == 7
    assert lib.bp_rope(None, None, 0, None, None, 1, 1, 2, None, None, None, 0.0, 0) == 7
    assert lib.bp_kv4_append(None, None, 0, None, None, None, 1, None, None, None, None, 0.0) == 7
    assert lib.bp_kv4_read(None, None, 0, None, None, 1, None, None) == 7
    assert lib.bp_kv4_attention(None, None, 0, None, None) == 7
    assert lib.bp_paged_last_error(None) == b""
    assert lib.bp_kv4_pool_bytes(None) == 0
    lib.bp_paged_destroy(None)
    import torch
    if not torch.cuda.is_available():
        with pytest.raises(bp.CudaError):
            bp.PagedContext()
        h = C.c_void_p()
        assert lib.bp_paged_create(0, C.byref(h)) == 5 and h  # set even on failure: the message
        assert b"no CUDA device" in lib.bp_paged_last_error(h)
        assert lib.bp_paged_status(h, None) == 5
        lib.bp_paged_destroy(h)


@pytest.mark.parametrize("gain", [0.0, 1e-7, 1e-4, 1.0, 300.0, 6e4, 1e6])
@pytest.mark.parametrize("shift", [0.0, 1.0, -30.0])
def test_every_value_of_a_block_is_an_f16_number_and_near_its_own(gain, shift):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((400, 128)) * gain + shift * gain).astype(np.float32)
    q, d, m = R.quantise(x)
    v = R.dequantise(q, d, m)
    assert np.isfinite(v).all() and np.array_equal(v, v.astype(np.float16).astype(np.float64))
    b = np.clip(x, -64512, 64512).reshape(400, 4, 32).astype(np.float64)
    top = np.abs(b).max(-1) * 65 / 64
    u = np.maximum(2.0 ** (np.floor(np.log2(np.where(top > 0, top, 1))) - 10), 2.0 ** -24)
    # half a step, half a unit that m is off, and fifteen halves by which d is: the largest code cuts there
    bound = np.maximum(d.astype(np.float64) / 2, 0) + 8 * u
    assert (np.abs(v.reshape(b.shape) - b) <= bound[..., None] * (1 + 1e-6)).all()
