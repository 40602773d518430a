"""The INT8 block's kernels against committed bits and, for the attention, its formula.

The bits (golden/block_*.npz, written by golden/make_block_golden.py) come from a build that
was compared bit for bit with the reference's own kernels; the operands are made by integer
arithmetic (block_inputs.py), so nothing of the reference is needed here."""
from pathlib import Path

import block_inputs
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
GOLDEN = Path(__file__).resolve().parent / "golden"


def same(name, out):
    golden = np.load(GOLDEN / f"{name}.npz")
    assert set(golden.files) == set(out)
    for key, t in out.items():
        assert np.array_equal(t.cpu().numpy(), golden[key]), key


@pytest.mark.parametrize("name", list(block_inputs.ATTENTION))
def test_attention_reproduces_golden(device, name):
    same(f"block_attention_{name}", block_inputs.run_attention(name, device))


@pytest.mark.parametrize("name", list(block_inputs.QKV))
def test_qkv_reproduces_golden(device, name):
    """Codes, scales and anchors, few and many rows; shared offsets make an anchor fire."""
    out = block_inputs.run_qkv(name, device)
    same(f"block_qkv_{name}", out)
    assert (out["anchors"] >= 0).any() == (name == "many")


def test_gelu_epilogue_reproduces_golden(device):
    same("block_gelu", block_inputs.run_gelu(device))


@pytest.mark.parametrize("name", list(block_inputs.ATTENTION))
def test_attention_against_its_formula(device, name):
    """softmax(Q K^T) V in 64 bits with every scale where it belongs: Q's of row r of a
    128-row block at 8 (r // 32) + r % 8 of 32, K's at (r % 8) // 2 of 4.

    The bound, per value: a weight is a whole number of 0 .. 255 of its 128-key block's
    largest, off by 1/2; the blocks' sums count those (the last block's the unrounded ones);
    a block with the largest b counts 2^(b - row's largest).  Then half a step of BF16, and
    1e-5 of the scores and weights for FP32, whose values below 2^-126 are flushed: a block that
    counts less adds up to 128 weights of 255 times codes of 127, over a sum of 255 at least,
    times a scale below 2^-6, less than 2^-126 2^14 2^-6 in all."""
    packed, start = block_inputs.attention(name, device)
    m, heads, kv_heads = packed.q.shape[2], packed.q.shape[1], packed.k.shape[1]
    got = block_inputs.run_attention(name, device)["out"].view(torch.bfloat16)[0]
    r = torch.arange(m, device=device)
    qs = packed.q_scale[0][:, r // 128 * 32 + r % 128 // 32 * 8 + r % 8].double()
    ks = packed.k_scale[0][:, r // 128 * 4 + r % 8 // 2].double()
    order = torch.tensor([0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15], device=device)
    v = torch.empty((kv_heads, 128, packed.v.shape[1] // 16, 16), dtype=torch.float64, device=device)
    v[..., order] = packed.v.view(kv_heads, 128, -1, 16).double()
    v = v.view(kv_heads, 128, -1)[..., :m].transpose(1, 2) * packed.v_scale.view(kv_heads, 1, 128).double()
    for h in range(heads):
        g = h // (heads // kv_heads)
        s = (packed.q[0, h].double() * qs[h][:, None]) @ (packed.k[0, g].double() * ks[g][:, None]).T * 128 ** -0.5
        want = s.softmax(-1) @ v[g]
        weights = 255 * torch.exp(s - s.amax(1, keepdim=True))
        off_n, off_d, blocks = torch.zeros_like(want), torch.zeros_like(want[:, :1]), range(0, m, 128)
        for j in blocks:
            share = torch.exp(s[:, j:j + 128].amax(1, keepdim=True) - s.amax(1, keepdim=True))
            off_n += 0.5 * share * v[g, j:j + 128].abs().sum(0)
            off_d += 0.5 * share * 128 * (j != blocks[-1])
        total = weights.sum(1, keepdim=True)
        fp32 = 1e-5 * (1 + s.abs().amax(1, keepdim=True)) * (s.softmax(-1) @ v[g].abs())
        bound = (off_n + want.abs() * off_d) / (total - off_d).clamp_min(255) + want.abs() * 2.0 ** -8 + fp32 + 2.0 ** -118
        rows = slice(start * 128, None)
        err = (got[h].double() - want).abs()[rows]
        assert torch.all(err <= bound[rows]), float((err / bound[rows]).max())
        assert bound[rows].mean() < want[rows].abs().mean(), "the bound says something"
