"""What the tests of the 16-bit products share: ragged groups, inputs, the formulas in 64 bits, and how far a
result may be from them.

A sum of K exact products (16-bit operands: each product is exact in FP32) takes at most K + 16 FP32 roundings,
and matrix instructions may cut instead of rounding: (K + 16) 2^-23 of sum |x w|.  The result rounds once: 2^-11
(FP16; below 2^-14 by 2^-25) or 2^-8 (BF16) of its size."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -23
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -149}
GUARD = -77.0


def torch_type(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


class Inputs:
    """Device tensors of normal values and their float64 copies; `shift` elements into their buffers."""

    def __init__(self, torch, dtype, seed=0, shift=0):
        self.torch, self.dtype, self.shift = torch, torch_type(torch, dtype), shift
        self.rng = np.random.default_rng(seed)

    def make(self, *shape, std=1.0):
        n = int(np.prod(shape))
        v = self.rng.standard_normal(n + self.shift).astype(np.float32) * std
        t = self.torch.from_numpy(v).to("cuda").to(self.dtype)[self.shift:].reshape(shape)
        return t, t.double().cpu().numpy()

    def out(self, *shape, dtype=None):
        """A result between guards: (the tensor, a check that the guards are whole)."""
        n = int(np.prod(shape))
        whole = self.torch.full((n + self.shift + 8,), GUARD, dtype=dtype or self.dtype, device="cuda")

        def check():
            h = whole.double().cpu().numpy()
            assert np.all(h[:self.shift] == GUARD) and np.all(h[self.shift + n:] == GUARD), "past the end"
        return whole[self.shift:self.shift + n].reshape(shape), check


def offsets_of(torch, counts, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def sums(x, w):
    """(x w^T, its absolute sums) in float64."""
    return x @ w.T, np.abs(x) @ np.abs(w).T


def sum_error(k, size):
    return (k + 16) * U * size


def close(got, want, err, dtype, what=""):
    """|got - want| within `err` and the one rounding to `dtype`."""
    got = np.asarray(got, np.float64)
    tol = err + HALF[dtype] * (np.abs(want) + err) + TINY[dtype]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[0].tolist(), got[bad][0], want[bad][0], tol[bad][0])


def silu_parts(g):
    """(s, g s) of a gate, in float64."""
    s = 1.0 / (1.0 + np.exp(-np.clip(g, -700, 700)))
    return s, g * s
