"""GPU tests of layer steps over the 4-bit cache that take the prompt kernel, and of the whole
layer (attention and MLP) against the library's own operations composed."""
import numpy as np
import pytest

import sib200
from test_gpu_kv4 import DIMS, DIMS128, expected_attn_step, up

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def composed_mlp(ctx, layer, dims, h):
    """h + down(silu(gate) * up) of rows h, each operation by its own entry point."""
    T, H = h.shape
    inner = dims["intermediate"]
    hq, hd = torch.zeros(T, H, dtype=torch.int8, device="cuda"), torch.zeros(T, H // 32, dtype=torch.int16, device="cuda")
    aq, ad = torch.zeros(T, inner, dtype=torch.int8, device="cuda"), torch.zeros(T, inner // 32, dtype=torch.int16, device="cuda")
    y, norm = torch.zeros(T, H, device="cuda"), up(layer.host()["norm2"])
    torch.cuda.synchronize()
    ctx.rmsnorm_q8(h, norm, T, H, dims["rms_eps"], None, hq, hd)
    ctx.gateup_q8(layer.matrix(2), layer.matrix(3), hq, hd, T, aq, ad)
    ctx.matmul(layer.matrix(4), aq, ad, T, None, y)
    ctx.sync()
    return h + y


@pytest.mark.parametrize("dims", [DIMS, DIMS128])
def test_steps_of_prompts_and_whole_layers(dims):
    """A prompt long enough for the prompt kernel, then one beside single tokens, in the
    attention mode against the composed formulas (the bar of the other step tests: one
    flipped Q8 code moves a row by about 1 / 127 of one input's share) and in the full mode
    against the MLP of that step's own output.  There the sums h may differ in their
    last bit, so of a row's thousands of Q8 codes a few may flip, each by 1 / 127 of one of
    thousands of inputs: 2e-4 of the row, 1e-3 for two dozen."""
    ctx = sib200.Context(0, max_positions=1024, rope_theta=1e6, head_dim=dims["head_dim"])
    layer = ctx.layer_synth(dims, 41)
    D, hkv, H = dims["head_dim"], dims["n_kv_heads"], dims["hidden"]
    kv = ctx.kv4(dims, 4, 1024, 110, 32)
    want_kv = [(np.zeros((1024, hkv, D)), np.zeros((1024, hkv, D))) for _ in range(4)]
    g = torch.Generator("cuda").manual_seed(42)
    for runs in ([(0, 0, 801)], [(0, 801, 1), (1, 0, 777), (2, 0, 3)], [(0, 802, 1), (3, 0, 1), (1, 777, 2)]):
        T = sum(r[2] for r in runs)
        x, y, z = torch.randn(T, H, device="cuda", generator=g), torch.zeros(T, H, device="cuda"), torch.zeros(T, H, device="cuda")
        torch.cuda.synchronize()
        layer.step_dev(kv, x, runs, y)
        layer.step_dev(kv, x, runs, z, sib200.SI_LAYER_FULL)
        ctx.status()
        got, want = y.cpu().numpy(), expected_attn_step(ctx, layer, dims, x, want_kv, runs)
        e = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
        assert e.max() < 1e-2, (runs, e.argmax(), e.max())
        full = composed_mlp(ctx, layer, dims, x + y)
        e = ((z - full).norm(dim=1) / (full - x).norm(dim=1)).max().item()
        assert e < 1e-3, (runs, e)
    kv.free()
    layer.free()
    ctx.close()
