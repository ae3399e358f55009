"""verify_tokens at the ends of its numbers: rows of the lowest value, logits and temperatures near the types' limits.
The reference and its tolerance (none: tokens are whole numbers) are those of ``test_gpu_verify``."""
import ctypes

import numpy as np
import pytest
import torch

from commitllm_b200 import _lib
from commitllm_b200 import decode as D
from tests import test_gpu_verify as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [11, 5000, 70001])
def test_verify_rows_of_the_lowest_value(ctx, dtype, V, with_probs):
    """What is allowed sits at the type's lowest value, the usual mask: it is drawn from like any other row."""
    S, k = 8, 2
    rng = np.random.default_rng(V)
    low = torch.finfo(base.DT[dtype]).min
    logits = torch.full((S, k + 1, V), low, device="cuda").to(base.DT[dtype])
    logits[2:, :, ::3] = -torch.inf                  # some ruled out for good
    logits[4:, 0, 5] = 1.0                           # one row with a likely token, the next without
    logits[6:, 1] = logits[6:, 1] / 2                # and one at half of the lowest value
    u = (np.arange(S * (k + 1)).reshape(S, k + 1) * 0.6180339887 + 0.0123457) % 1.0
    temperature = np.array([1.0, 0.7, 1.0, 3.0, 0.5, 1.0, 2.0, 0.0], np.float32)
    probs = None
    drafts = rng.integers(0, V, (S, k)).astype(np.int32)
    if with_probs:
        probs = torch.softmax(torch.tensor(rng.standard_normal((S, k, V)).astype(np.float32), device="cuda"), -1)
    else:
        # what is drawn first without drafts, so that some are kept
        want, _ = base.plain(logits.double().cpu().numpy(), drafts, u, temperature)
        drafts[::2, 0] = want[::2, 0]
    base.check(ctx, logits, drafts, u, temperature, probs)


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("t", [1e-45, 1e-42, 3e-39, 1e-36, 1e30, 1e34, 1e36, 1e37, 1e38, 3e38])
def test_verify_temperatures_at_the_types_ends(ctx, t, with_probs):
    """Logits that differ by a few temperatures, however small or large that is."""
    S, k, V = 32, 2, 3001
    rng = np.random.default_rng(23)
    t = float(np.float32(t))
    spread = min(4.0 * t, 3.3e38)
    l = np.clip(rng.uniform(-spread, spread, (S, k + 1, V)), -3.4e38, 3.4e38).astype(np.float32)
    l[:, :, 1::7] = np.finfo(np.float32).min
    u = rng.random((S, k + 1))
    temperature = np.full(S, t, np.float32)
    logits = torch.tensor(l, device="cuda")
    drafts = rng.integers(0, V, (S, k)).astype(np.int32)
    probs = None
    if with_probs:
        probs = torch.softmax(torch.tensor(rng.standard_normal((S, k, V)).astype(np.float32), device="cuda"), -1)
    else:
        want, _ = base.plain(l.astype(np.float64), drafts, u, temperature)
        drafts[::2, 0] = want[::2, 0]
    base.check(ctx, logits, drafts, u, temperature, probs)


def test_verify_workspace_is_what_the_library_asks_for(ctx):
    for S, k, V in ((1, 0, 1), (3, 4, 128256), (64, 7, 152064), (700, 1, 2), (1, 1, 1 << 20)):
        out = ctypes.c_size_t()
        assert _lib.lib().vc_verify_tokens_workspace(ctx.handle, S, k, V, ctypes.byref(out)) == _lib.VC_OK
        assert out.value == S * (k + 1) * D._VERIFY_ROW_BYTES
