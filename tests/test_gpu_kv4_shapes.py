"""GPU tests of the 4-bit cache's attention: odd numbers of heads, where the partial
sums of split keys have an odd number of slots, and scores of which one lies far above
the others."""
import numpy as np
import pytest

import sib200
from test_gpu_kv4 import Cache, up

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(7, 1, 128), (7, 1, 64), (1, 1, 128), (5, 1, 64), (9, 3, 128)])
def test_odd_heads_decode_with_many_splits(si_ctx, heads):
    """Lengths whose split counts lie above eight, odd and even ones, alone and in threes."""
    lens = [6200, 7000, 8200, 20000]
    c = Cache(si_ctx, heads, len(lens), 20000, 64, seed=31)
    c.random([(s, 0, n) for s, n in enumerate(lens)])
    calls = [[(s, n - 1, 1)] for s, n in enumerate(lens)]
    calls += [[(0, 6198, 1), (1, 6998, 1), (2, 8000, 1)]]
    for runs in calls:
        q = c.rng.standard_normal((len(runs), heads[0], heads[2]))
        c.check(c.attend(q, runs), q, runs)
    c.kv.free()


@pytest.mark.parametrize("B", [7, 5, 1])
def test_odd_batch_with_device_lengths(B):
    """A captured-form step over a long cache (up to 63 splits) against the step with
    host runs: one flipped Q8 code of the attention output moves a row by about 1 / 127
    of one input's share, the bar of the other step tests."""
    D = 128
    dims = dict(hidden=7 * D, n_q_heads=7, n_kv_heads=1, head_dim=D, intermediate=0,
                rope_theta=1e6, rms_eps=1e-6)
    L = 8192
    ctx = sib200.Context(0, max_positions=L, rope_theta=1e6, head_dim=D)
    layer = ctx.layer_synth(dims, 33)
    rng = np.random.default_rng(34)
    lens = [int(n) for n in rng.integers(1, L - 1, B)]
    lens[0] = L - 1
    T = sum(lens)
    g = torch.Generator("cuda").manual_seed(35)
    k, v = (torch.randn(T, 1, D, device="cuda", generator=g) for _ in range(2))
    x = torch.randn(B, 7 * D, device="cuda", generator=g)
    ya, yb = torch.zeros_like(x), torch.zeros_like(x)
    torch.cuda.synchronize()
    kvs = [ctx.kv4(dims, B, L, B * L // 64, 64) for _ in range(2)]
    for kv in kvs:
        kv.append(k, v, [(s, 0, n) for s, n in enumerate(lens)])
    layer.step_dev(kvs[0], x, [(s, n, 1) for s, n in enumerate(lens)], ya)
    kvs[1].reserve([(s, n, 1) for s, n in enumerate(lens)])
    st = ctx.decode_state([n + 1 for n in lens], L)
    layer.decode_state_dev(kvs[1], x, st, yb)
    ctx.status()
    a, b = ya.cpu().numpy(), yb.cpu().numpy()
    for t in range(B):
        assert np.linalg.norm(a[t] - b[t]) <= 1e-2 * np.linalg.norm(a[t]), (t, lens[t])
    ctx.close()


@pytest.mark.parametrize("heads", [(7, 1, 128), (7, 1, 64), (5, 1, 128), (9, 3, 64)])
@pytest.mark.parametrize("prefix,count", [(2000, 201), (3000, 255), (4000, 129), (1000, 501)])
def test_odd_heads_prompts_with_splits(si_ctx, heads, prefix, count):
    """Prompts of few row tiles, whose keys are split, odd in tokens and heads; with a
    second prompt of another length in the same call."""
    c = Cache(si_ctx, heads, 2, prefix + count, 48, seed=32)
    c.random([(0, 0, prefix + count), (1, 0, 331)])
    for runs in ([(0, prefix, count)], [(1, 200, 131), (0, prefix, count)]):
        q = c.rng.standard_normal((sum(r[2] for r in runs), heads[0], heads[2]))
        c.check(c.attend(q, runs), q, runs, every=29)
    c.kv.free()


@pytest.mark.parametrize("nats", [8, 10, 12, 17])
@pytest.mark.parametrize("heads,prefix,count", [
    ((28, 4, 128), 0, 2048), ((16, 2, 128), 7580, 612), ((16, 2, 64), 7580, 612),
    ((16, 2, 128), 40000, 612), ((12, 2, 128), 7900, 131), ((12, 2, 128), 8000, 2)])
def test_a_first_key_far_above_the_others(si_ctx, heads, prefix, count, nats):
    """Position 0 takes much of every row's weight and holds small values, as the first
    token of a text does: the others, each of 2^-12 to 2^-25 of its weight, make the
    output.  In one split of the keys, in many, and token by token."""
    hq, hkv, D = heads
    n = prefix + count
    c = Cache(si_ctx, heads, 1, n, 64, seed=36)
    k, v = (c.rng.standard_normal((n, hkv, D)) for _ in range(2))
    u = np.sign(c.rng.standard_normal(D))
    k[0] = u
    v[0] *= 0.05
    c.append([(0, 0, n)], k, v)
    # u.q / sqrt(D) is the sink's score: noise of one nat about the given number
    q = c.rng.standard_normal((count, hq, D)) + nats / np.sqrt(D) * u
    runs = [(0, prefix, count)]
    c.check(c.attend(q, runs), q, runs, every=199)
    c.kv.free()


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("count", [12, 13, 15, 16, 17])
def test_short_runs_on_many_positions(si_ctx, count, exact):
    """Runs on both sides of the fewest tokens of either prompt kernel, with enough work
    for them, alone and beside a longer one."""
    heads = (64, 8, 128)
    c = Cache(si_ctx, heads, 2, 6100, 64, seed=37)
    c.random([(0, 0, 6100), (1, 0, 2000)])
    si_ctx.set_exact_attention(exact)
    try:
        for runs in ([(0, 6100 - count, count)], [(0, 6001, count), (1, 1900, 40), (0, 3000, 13)]):
            q = c.rng.standard_normal((sum(r[2] for r in runs), heads[0], heads[2]))
            c.check(c.attend(q, runs), q, runs, every=6)
    finally:
        si_ctx.set_exact_attention(False)
    c.kv.free()


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("prefix,where", [(4100, 57), (4100, 0), (20, 57)])
def test_values_that_are_no_numbers_reach_only_later_rows(si_ctx, heads, prefix, where, what, exact):
    """One block of one head's V of position prefix + where is no number: the rows before it
    and the other KV head's keep their results, in every kernel."""
    hq, hkv, D = heads
    c = Cache(si_ctx, heads, 1, prefix + 100, 32, seed=38)
    c.random([(0, 0, prefix + 100)])
    one = np.ones((1, hkv, D), np.float32)
    bad = one.copy()
    bad[0, 1, 32:64] = what
    kd, vd = up(one), up(bad)
    torch.cuda.synchronize()
    c.kv.append(kd, vd, [(0, prefix + where, 1)])
    q = c.rng.standard_normal((100, hq, D))
    si_ctx.set_exact_attention(exact)
    try:
        got = c.attend(q, [(0, prefix, 100)])
    finally:
        si_ctx.set_exact_attention(False)
    assert np.isfinite(got[:where]).all()
    if where:
        c.check(got[:where], q[:where], [(0, prefix, where)], every=19)
    assert np.isfinite(got[:, :hq // 2]).all()
    assert np.isnan(got[where:, hq // 2:, 32:64]).all()


@pytest.mark.parametrize("heads,prefix,count", [((28, 4, 128), 500, 200), ((14, 2, 64), 3200, 211),
                                                ((16, 2, 128), 7580, 612)])
@pytest.mark.parametrize("qscale", [0.0, 1e-3, 6.0, 30.0])
def test_sharp_and_flat_softmax_of_prompts(si_ctx, heads, prefix, count, qscale):
    c = Cache(si_ctx, heads, 1, prefix + count, 64, seed=39)
    c.random([(0, 0, prefix + count)])
    runs = [(0, prefix, count)]
    q = c.rng.standard_normal((count, heads[0], heads[2])) * qscale
    c.check(c.attend(q, runs), q, runs, every=37)
    c.kv.free()


@pytest.mark.parametrize("vscale", [1e-5, 1e-3, 0.01, 0.1, 1.0, 4.0, 30.0, 300.0, 3000.0, 4e4])
@pytest.mark.parametrize("heads,prefix,count,times", [
    ((12, 2, 128), 8000, 2, 1), ((12, 2, 128), 7900, 131, 1),
    ((64, 8, 128), 2100, 12, 6), ((56, 8, 64), 2100, 12, 6)])
def test_a_first_key_far_above_values_of_any_size(si_ctx, heads, prefix, count, times, vscale):
    """As above, with values of other sizes, whose scales must not take the bits of the
    small probabilities: in many splits, in a prompt, and in a batch that fills the GPU
    with a split or two of each token."""
    hq, hkv, D = heads
    n = prefix + count
    c = Cache(si_ctx, heads, 1, n, 64, seed=40)
    k, v = (c.rng.standard_normal((n, hkv, D)) for _ in range(2))
    u = np.sign(c.rng.standard_normal(D))
    k[0] = u
    v *= vscale
    v[0] *= 1e-6
    c.append([(0, 0, n)], k, v)
    q = c.rng.standard_normal((count * times, hq, D)) + 13 / np.sqrt(D) * u
    runs = [(0, prefix, count)] * times
    got = c.attend(q, runs)
    c.check(got[:count], q[:count], runs[:1], every=29)
    c.check(got[-count:], q[-count:], runs[:1], every=29)
    c.kv.free()
