"""GPU: paged attention and append where small differences count, against the
definitions in 64 bits; the helpers and their bounds are those of the tests of
the ordinary cases."""

import pytest
import torch

from preemptlm_b200 import ops

from .test_gpu_paged_attention import DEV, attend64, make_cache, make_table, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,heads,group", [(64, 2, 8), (128, 2, 5), (128, 1, 16), (256, 2, 8), (256, 1, 16)])
def test_probabilities_keep_sixteen_bits(bits, D, heads, group):
    """Pairs of tokens with opposite values and nearly equal scores: the output is the small difference of their
    probabilities.  Bound: one rounding of the output (2^-8 of it), and 2^-15 of the sum of probability * |v|: sixteen
    bits of a probability (2^-17), and below 2e-5 for fp32 scores (|score| < 0.1), exponential and sums of up to 64
    tokens."""
    lengths, page = [2, 4, 16, 34, 64], 16
    table, total = make_table(lengths, page, 1)
    cache = make_cache(total, heads, page, D, bits, 2)
    cache.v[:, :, 1::2] = (-cache.v[:, :, 0::2].float()).to(cache.v.dtype)
    q = rand((len(lengths), heads * group, D), 5, 0.01)
    got = ops.paged_attention(cache, q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    ref, mag = attend64(cache, q, table, lengths)
    err = (got.double() - ref).abs()
    bound = ref.abs() * 2.0 ** -8 + mag * 2.0 ** -15
    assert bool((err <= bound).all()), float((err / bound).max())
