"""The short roots and quotients of AdamW with 8-bit moments (csrc/adamw.hip), bit for bit against numpy's, where they could go
wrong: the root of every value of two octaves (a root's mantissa goes by its argument's modulo 4), divisors whose mantissa is all
ones, or nearly, under numerators of every mantissa.  What a parameter of 0 moves by with a step size of 1 is the quotient itself."""
import numpy as np
import pytest
import torch

from test_adamw_gpu import BLOCK, step_and_check

pytestmark = pytest.mark.gpu

STEP = 200  # 1 - 0.5^200 is 1 in fp32: neither root nor step size is changed by the bias corrections
HYPER = dict(lr=1.0, beta1=0.5, beta2=0.5, weight_decay=0.0)
TOP = torch.tensor(448.0).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("octave", [0, 1])
@pytest.mark.parametrize("numerator", ["below the root", "one"])
def test_roots_of_every_mantissa(octave, numerator):
    """v' = (top scale)^2 / 2 + g^2 / 2: the first term near the block's base, the second 0 .. 255 units in its last place.  With
    numerators just below the root (quotients in [0.98, 1), whose units are as fine as the root's) another root is another quotient."""
    f, unit, apart = np.float32, 2.0 ** (octave - 23), 248  # (neighbouring blocks overlap by more than the base's own roundings)
    k = np.arange(-(-(1 << 23) // apart) + 1)
    base = 2.0 ** octave + k * apart * unit
    k, base = k[base < 2.0 ** (octave + 1) + 16 * unit], base[base < 2.0 ** (octave + 1) + 16 * unit]
    n = len(k) * BLOCK
    vs = (np.sqrt(2 * (base - 4 * unit)) / 448).astype(f)
    g = np.tile(np.sqrt(2 * np.arange(BLOCK) * unit), len(k)).astype(f)
    r0 = (vs * f(448))[:, None]
    v1 = ((r0 * r0) * f(0.5) + ((g * f(0.5)) * g).reshape(-1, BLOCK)).reshape(-1)
    hit = np.unique(v1[(v1 >= 2.0 ** octave) & (v1 < 2.0 ** (octave + 1))].view(np.uint32))
    assert len(hit) == 1 << 23  # every one
    ms = (2 * (np.sqrt(base) * 0.98 if numerator != "one" else np.ones(len(k))) / 448).astype(f)
    codes = TOP.expand(n).clone()
    step_and_check([[torch.zeros(n), torch.from_numpy(g), codes, codes.clone(), torch.from_numpy(ms), torch.from_numpy(vs)]], STEP, 8,
                   hyper=dict(HYPER, eps=0.0))


@pytest.mark.parametrize("eps", ["0x1.fffffep-10", "0x1.fffffcp-10", "0x1.fffffap-10", "0x1.0d3226p-10", "0x1.0p-10"])
def test_divisors_at_the_end_of_their_octave(eps):
    """g of every mantissa, so small that the root (below 2^-43) vanishes beside eps: the divisor is eps"""
    n, eps = 1 << 23, float.fromhex(eps)
    g = (np.arange(n, dtype=np.int32) + ((127 - 44) << 23)).view(np.float32).copy()
    g[1::2] *= -1
    g = np.concatenate([g, -g])
    assert np.all(np.sqrt(0.5 * g.astype(np.float64) ** 2) < eps * 2.0 ** -25) and np.float32(eps) == eps
    zero = torch.zeros(2 * n).to(torch.float8_e4m3fn)
    none = torch.zeros(2 * n // BLOCK)
    step_and_check([[torch.zeros(2 * n), torch.from_numpy(g), zero, zero.clone(), none, none.clone()]], STEP, 8, hyper=dict(HYPER, eps=eps))
