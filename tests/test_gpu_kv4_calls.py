"""GPU tests of calls on the 4-bit cache that are refused."""
import pytest

import sib200

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_a_step_that_lacks_memory_takes_no_pages():
    """Two million tokens of the 72B dims want 375 GB of workspace."""
    dims = dict(hidden=8192, n_q_heads=64, n_kv_heads=8, head_dim=128, intermediate=0,
                rope_theta=1e6, rms_eps=1e-6)
    ctx = sib200.Context(0, max_positions=8192, rope_theta=1e6, head_dim=128)
    layer = ctx.layer_synth(dims, 2)
    kv = ctx.kv4(dims, 256, 8192, 512, 4096)
    x, y = torch.randn(1, 8192, device="cuda"), torch.zeros(1, 8192, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(sib200.SiError) as e:
        layer.step_dev(kv, x, [(s, 0, 8192) for s in range(256)], y)
    assert e.value.status == sib200.SI_ERR_OOM
    assert kv.free_pages() == 512 and kv.pages(0) == []
    layer.step_dev(kv, x, [(3, 0, 1)], y)
    ctx.status()
    assert kv.free_pages() == 511 and torch.isfinite(y).all()
    ctx.close()


@pytest.mark.parametrize("n_q_heads", [0, -8])
def test_attention_without_query_heads_is_refused(si_ctx, n_q_heads):
    dims = dict(hidden=1024, n_q_heads=8, n_kv_heads=8, head_dim=128, intermediate=0)
    kv = si_ctx.kv4(dims, 1, 4096, 64, 64)
    kv.reserve([(0, 0, 4096)])
    q, out = torch.randn(64, 1024, device="cuda"), torch.zeros(64, 1024, device="cuda")
    torch.cuda.synchronize()
    for runs in ([(0, 300, 1)], [(0, 4032, 64)]):
        with pytest.raises(sib200.SiError) as e:
            si_ctx.attention_kv4(kv, dict(dims, n_q_heads=n_q_heads), q, runs, out)
        assert e.value.status == sib200.SI_ERR_INVALID
    si_ctx.attention_kv4(kv, dims, q, [(0, 4032, 64)], out)
    si_ctx.status()
    assert torch.isfinite(out).all()
    kv.free()


def test_pages_of_four_gigabytes_are_refused(si_ctx):
    """Whose heads lie at offsets past 32 bits; the page length below is taken."""
    dims = dict(hidden=1024, n_q_heads=8192, n_kv_heads=8192, head_dim=128, intermediate=0)
    assert sib200.kv4_page_bytes(dims, 4096) > 1 << 32
    small = torch.zeros(1024, dtype=torch.uint8, device="cuda")  # not touched by the creation
    with pytest.raises(sib200.SiError) as e:
        si_ctx.kv4(dims, 1, 4096, 1, 4096, small.data_ptr())
    assert e.value.status == sib200.SI_ERR_INVALID
    si_ctx.kv4(dims, 1, 4096, 1, 2048, small.data_ptr()).free()


def test_a_pool_in_host_memory_is_refused(si_ctx):
    dims = dict(hidden=1024, n_q_heads=8, n_kv_heads=8, head_dim=128, intermediate=0)
    pool = torch.zeros(4 * sib200.kv4_page_bytes(dims, 16), dtype=torch.uint8)
    for p in (pool, pool.numpy(), pool.data_ptr()):
        with pytest.raises(sib200.SiError) as e:
            si_ctx.kv4(dims, 1, 64, 4, 16, p)
        assert e.value.status == sib200.SI_ERR_INVALID
    si_ctx.kv4(dims, 1, 64, 4, 16, pool.cuda()).free()
