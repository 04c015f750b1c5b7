"""Refusals of the decoder operators that need no GPU, at the edges of what their documentation allows."""

import pytest
import torch

import tilegym_b200 as tg
from tilegym_b200 import _lib

F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def _d(t):
    return _lib.desc(t)


def test_norm_refuses_a_sum_over_rows_that_are_still_read():
    """H may take the place of X or of the residual where their rows are dense: row t of H then lies on row t.  With a pitch,
    or shifted, it would lie on rows that other blocks have still to read."""
    L = _lib.lib()
    w, y, s = torch.zeros(256, dtype=BF), torch.zeros(4, 256, dtype=F8), torch.zeros(4, 2)
    memory = torch.zeros(4096, dtype=BF)
    dense, pitched, shifted = memory[:1024].view(4, 256), memory.view(8, 512)[:4, :256], memory[256:1280].view(4, 256)
    other = torch.zeros(4, 256, dtype=BF)

    def call(H, X, R, T=4):
        return L.tg_rms_norm_quant(_d(y[:T]), _d(s[:T]), _d(H), _d(X), _d(R), _d(w), 1e-6, 0.0, 0, 0)

    for X, R in ((pitched, other), (other, pitched), (shifted, other), (other, shifted), (dense, pitched)):
        assert call(dense, X, R) == -6, (X.stride(), R.stride())
    if not torch.cuda.is_available():  # these get as far as the device, which must not be given host memory
        for H, X, R, T in ((dense, dense, other, 4), (dense, other, dense, 4), (dense, dense, dense, 4), (other, pitched, shifted, 4),
                           (dense[:1], pitched[:1], other[:1], 1)):
            assert call(H, X, R, T) != -6
