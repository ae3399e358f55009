"""Host side of the decode-step operators: rope frequencies, and refusals that need no GPU."""
import ctypes
import math
import struct

import numpy as np
import pytest

from commitllm_b200 import _lib
from commitllm_b200 import commit as C
from commitllm_b200 import decode as D
from oracle import commit_oracle as O


@pytest.mark.parametrize("scaling", [None, "linear", "llama3"])
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_frequencies_equal_the_transcripts(scaling, dim):
    """The scalings that the KV transcript has: every f64 equal to the oracle's."""
    cfg = C.RopeConfig(theta=500000.0, scaling=scaling)
    inv, factor = D.rope_frequencies(cfg, dim)
    want = O.scaled_inv_freq(dim, 500000.0, O.RopeScaling(rope_type=scaling) if scaling else None)
    assert factor == 1.0
    assert np.array_equal(np.asarray(inv), np.asarray(want))


def test_yarn_frequencies():
    cfg = C.RopeConfig(theta=10000.0, scaling="yarn", factor=16.0, original_max_position_embeddings=4096)
    inv, factor = D.rope_frequencies(cfg, 128)
    plain = [10000.0 ** (-2 * i / 128) for i in range(64)]
    assert factor == 0.1 * math.log(16.0) + 1.0
    assert np.allclose(inv[:16], plain[:16], rtol=1e-15) and np.allclose(inv[-10:], np.asarray(plain[-10:]) / 16, rtol=1e-15)
    assert all(a >= b for a, b in zip(inv, inv[1:]))
    # between the ends: a pair that turns t times in the original length is part stretched
    i = 30
    lo = math.floor(128 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    s = (i - lo) / (hi - lo)
    assert 0 < s < 1 and inv[i] == pytest.approx(plain[i] * (1 - s) + plain[i] / 16 * s, rel=1e-15)
    assert D.rope_frequencies(cfg, 128, attention_factor=1.0)[1] == 1.0


@pytest.mark.parametrize("cfg,dim", [(C.RopeConfig(scaling="other"), 64), (C.RopeConfig(), 7), (C.RopeConfig(), 0),
                                     (C.RopeConfig(theta=0.0), 64), (C.RopeConfig(scaling="linear", factor=0.0), 64),
                                     (C.RopeConfig(theta=1.0, scaling="yarn"), 64),
                                     (C.RopeConfig(scaling="llama3", low_freq_factor=4.0), 64)])
def test_frequency_refusals(cfg, dim):
    with pytest.raises(ValueError):
        D.rope_frequencies(cfg, dim)


def test_entry_points_refuse_null_arguments():
    lib = _lib.lib()
    assert lib.vc_rope_append(None, None, 0, 0, None, None, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, 0,
                              1.0, 0) == _lib.VC_EINVAL
    assert lib.vc_paged_attention(None, None, 0, 0, 0, 0, None, 0, 0, 0, None, 1.0, None, None, None, 0) == _lib.VC_EINVAL
    out = ctypes.c_size_t()
    assert lib.vc_paged_attention_workspace(None, None, 0, 0, ctypes.byref(out)) == _lib.VC_EINVAL
    assert lib.vc_verify_tokens(None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, None, None, None, None, None, None,
                                0) == _lib.VC_EINVAL
    assert lib.vc_decode_call(0, 23, None) == _lib.VC_EINVAL
    assert lib.vc_decode_call(3, 0, b"") == _lib.VC_EINVAL
    assert lib.vc_decode_call(1, 15, bytes(120)) == _lib.VC_EINVAL
    assert lib.vc_decode_call(1, 16, bytes(128)) == _lib.VC_EINVAL
    assert lib.vc_verify_tokens_workspace(None, 0, 0, 0, ctypes.byref(out)) == _lib.VC_EINVAL


def packed_call(which, values):
    """A vc_decode_call of these arguments (ints, floats), the context a block of zeros that no check reads."""
    lib = _lib.lib()
    ctx = ctypes.create_string_buffer(4096)
    slots = struct.pack("q" * (len(values) + 1), ctypes.addressof(ctx),
                        *(v if isinstance(v, int) else struct.unpack("q", struct.pack("d", v))[0] for v in values))
    return lib.vc_decode_call(which, len(values) + 1, slots)


def test_packed_arguments_past_32_bits_are_refused():
    """32-bit arguments in 64-bit slots: a value that does not fit is an error, not its low half.  Empty calls, which
    return before they touch a GPU."""
    k, v = (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)(512)
    d = _lib.KvDesc()
    d.n_layers = d.n_kv_heads = 1
    d.head_dim, d.dtype, d.n_seqs, d.block_size, d.max_blocks_per_seq = 64, _lib.VC_DTYPE_BF16, 2, 16, 4
    d.stride_page, d.stride_row, d.stride_head, d.cache_elems, d.block_tables = 1024, 64, 64, 8192, 256
    d.k_layers, d.v_layers = (ctypes.cast(p, ctypes.POINTER(ctypes.c_void_p)) for p in (k, v))
    desc = ctypes.addressof(d)
    rope = [desc, 0, 0, 256, 0, 1, 256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 64, 64, 256, 64, 1.0, 0]
    attend = [desc, 0, 0, 1, 1, 256, 64, 64, 64, 256, 0.125, 256, 0, 256, 1 << 20]
    verify = [0, 1, 100, 256, _lib.VC_DTYPE_F32, 200, 100, 0, 0, 0, 256, 256, 256, 256, 256, 256, 1 << 20]
    for which, good, narrow in ((_lib.VC_CALL_ROPE_APPEND, rope, (1, 2, 5, 19, 21)),
                                (_lib.VC_CALL_PAGED_ATTENTION, attend, (1, 2, 3, 4)),
                                (_lib.VC_CALL_VERIFY_TOKENS, verify, (0, 1, 2, 4))):
        assert packed_call(which, good) == _lib.VC_OK
        for at in narrow:
            for off in (1 << 32, -(1 << 32), 1 << 40):
                bad = list(good)
                bad[at] += off
                assert packed_call(which, bad) == _lib.VC_EINVAL, (which, at, off)
                assert "32 bits" in _lib.last_error()


def test_rope_append_refuses_outputs_that_overlap():
    """Strides of q_out against every pair of rows, on the CPU: calls that pass the check stop at a NULL
    position array."""
    k, v = (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)(512)
    d = _lib.KvDesc()
    d.n_layers = d.n_kv_heads = 1
    d.head_dim, d.dtype, d.n_seqs, d.block_size, d.max_blocks_per_seq = 4, _lib.VC_DTYPE_BF16, 8, 16, 4
    d.stride_page, d.stride_row, d.stride_head, d.cache_elems, d.block_tables = 64, 4, 4, 512, 256
    d.k_layers, d.v_layers = (ctypes.cast(p, ctypes.POINTER(ctypes.c_void_p)) for p in (k, v))
    seen = set()
    for heads in (1, 2, 3, 5):
        for toks in (1, 2, 4):
            for hs in (0, 2, 4, -4, 5, 6, 8, 12, 16, 2 ** 62):
                for ts in (0, 3, 4, -8, 6, 8, 10, 12, 16, 20, -2 ** 63):
                    rows = [range(h * hs + t * ts, h * hs + t * ts + 4) for h in range(heads) for t in range(toks)]
                    starts = sorted(r.start for r in rows)
                    want = any(b - a < 4 for a, b in zip(starts, starts[1:]))
                    got = packed_call(_lib.VC_CALL_ROPE_APPEND,
                                      [ctypes.addressof(d), 0, toks, 0, 0, heads, 256, 4, 4, 256, ts, hs, 256, 4, 4, 256, 4, 4,
                                       256, 4, 1.0, 0])
                    assert got == _lib.VC_EINVAL
                    assert ("overlap" in _lib.last_error()) == want, (heads, toks, hs, ts)
                    seen.add(want)
    assert seen == {False, True}
    d.v_layers = d.k_layers
    assert packed_call(_lib.VC_CALL_ROPE_APPEND, [ctypes.addressof(d), 0, 1, 0, 0, 1, 256, 4, 4, 256, 4, 4, 256, 4, 4, 256, 4, 4,
                                                  256, 4, 1.0, 0]) == _lib.VC_EINVAL
    assert "overlap" in _lib.last_error()


def test_rope_append_refuses_tokens_past_its_counters():
    """A token's chunks are counted in 32 bits: 2^30 elements are the most, empty calls on the CPU."""
    k, v = (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)(512)
    d = _lib.KvDesc()
    d.n_layers = d.n_kv_heads = 1
    d.head_dim, d.dtype, d.n_seqs, d.block_size, d.max_blocks_per_seq = 2, _lib.VC_DTYPE_BF16, 1, 16, 4
    d.stride_page, d.stride_row, d.stride_head, d.cache_elems, d.block_tables = 32, 2, 2, 512, 256
    d.k_layers, d.v_layers = (ctypes.cast(p, ctypes.POINTER(ctypes.c_void_p)) for p in (k, v))
    for heads, want in ((2 ** 29 - 2, _lib.VC_OK), (2 ** 29 - 1, _lib.VC_ENOTSUP), (2 ** 31 - 1, _lib.VC_ENOTSUP)):
        assert packed_call(_lib.VC_CALL_ROPE_APPEND, [ctypes.addressof(d), 0, 0, 256, 0, heads, 256, 2, 2, 256, 0, 2, 256, 2, 2, 256,
                                                      2, 2, 256, 2, 1.0, 0]) == want
