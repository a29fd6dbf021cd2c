"""GPU: the attention block over long prompts and the decoder layer over a prompt and
captured steps.  The 64-bit reference and its bounds are those of the block's tests."""

import pytest
import torch

from preemptlm_b200 import DecoderLayer, PagedAttention, PagedKVCache, Qwen3_xMoEWrapper, ops, rope_table
from preemptlm_b200.synthetic import LayerConfig, make_layer

from .test_gpu_decoder_layer import BF, DEV, F8, REL_L2, attention64, close, make, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,Hq,Hkv,D,page", [(BF, 256, 8, 2, 64, 16), (F8, 256, 4, 1, 128, 64), (BF, 512, 4, 2, 256, 8)])
@pytest.mark.parametrize("first", [0, 701])
def test_long_prompt(dtype, H, Hq, Hkv, D, page, first):
    """A prompt of 2301 tokens in one call, from the start or behind 701 cached tokens, through a table for 131072."""
    n = 2301 + first
    cache = PagedKVCache.empty(-(-n // page) + 3, Hkv, page, D, dtype, k_scale=0.02, v_scale=0.02)
    att = PagedAttention.from_weights(
        rand((H,), 1, 0.1) + 1, rand(((Hq + 2 * Hkv) * D, H), 2, 0.03), rand((H, Hq * D), 3, 0.03), cache, Hq,
        rope=rope_table(4096, 64, 1e4), q_norm=rand((D,), 4, 0.1) + 1, k_norm=rand((D,), 5, 0.1) + 1)
    table = torch.full((2, 131072 // page), -1, dtype=torch.int32, device=DEV)
    table[1, : -(-n // page)] = torch.randperm(-(-n // page), device=DEV, dtype=torch.int32,
                                               generator=torch.Generator(device=DEV).manual_seed(6))
    x, r = rand((n, H), 7), rand((n, H), 8, 2.0)
    pos = torch.arange(n, device=DEV, dtype=torch.int32)
    rows = torch.ones_like(pos)
    ops.device_status()
    got = [att(x[a:b], r[a:b], table, pos[a:b], rows[a:b]) for a, b in ((0, first), (first, n)) if a < b]
    assert ops.device_status() == 0
    ref, href = attention64(att, x, r)
    close(torch.cat([y for y, _ in got]), ref, 2.0 ** -4 if dtype == F8 else REL_L2)
    close(torch.cat([h for _, h in got]), href)


def test_decoder_layer_prompt_and_captured_steps():
    """Two sequences: their prompts in one call, then steps from a captured graph, padding among them; each call equals
    its parts, and the replayed steps the plain ones."""
    cfg = LayerConfig("layer-q8", 3, 512, 64, 4, 128, 128, 8, 64)
    block, _ = make_layer(cfg, device=DEV)
    moe = Qwen3_xMoEWrapper(block, "fp", "model.layers.0.mlp", 0)
    att = make(512, 8, 2, 64, 64, 16, 24, BF)
    layer = DecoderLayer(att, rand((512,), 30, 0.1) + 1, moe)
    table = torch.randperm(24, device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(3)).view(2, 12)
    lengths, steps = [150, 61], 5
    rows = torch.cat([torch.full((n,), b, dtype=torch.int32, device=DEV) for b, n in enumerate(lengths)])
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device=DEV) for n in lengths])
    x, r = rand((sum(lengths), 512), 31), rand((sum(lengths), 512), 32, 2.0)
    sx, sr = rand((steps, 3, 512), 33), rand((steps, 3, 512), 34, 2.0)
    step_rows = torch.tensor([0, -1, 1], dtype=torch.int32, device=DEV)  # the middle token is padding
    step_pos = torch.tensor([[lengths[0] + t, -1, lengths[1] + t] for t in range(steps)], dtype=torch.int32, device=DEV)

    def parts(x, r, pos, rows):
        a, h = att(x, r, table, pos, rows)
        y, h = ops.add_rms_norm(a, layer.post_norm, residual=h)
        return moe(y[None])[0], h

    want = [parts(x, r, pos, rows)] + [parts(sx[t], sr[t], step_pos[t], step_rows) for t in range(steps)]
    for c in (att.cache.k, att.cache.v):
        c.zero_()
    gx, gr, gp = sx[0].clone(), sr[0].clone(), torch.full((3,), -1, dtype=torch.int32, device=DEV)
    layer(gx, gr, table, gp, step_rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gh = layer(gx, gr, table, gp, step_rows)
    ops.device_status()
    got = [layer(x, r, table, pos, rows)]
    for t in range(steps):
        gx.copy_(sx[t])
        gr.copy_(sr[t])
        gp.copy_(step_pos[t])
        graph.replay()
        got.append((gy.clone(), gh.clone()))
    assert ops.device_status() == 0
    for (y, h), (y1, h1) in zip(got, want):
        assert torch.equal(y, y1) and torch.equal(h, h1)
    close(got[0][1], torch.cat([attention64(att, x[rows == b], r[rows == b])[0] + x[rows == b].double() + r[rows == b].double()
                                for b in range(2)]))
