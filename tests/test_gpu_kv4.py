"""GPU tests of the paged KV cache in 4 bits: written rows against the Q4_0 rule
bit for bit and byte for byte in the pool, attention against the formula in 64
bits (bounds derived in kv4_ref.py), page sharing, layer steps, captured steps,
and refusals."""
import numpy as np
import pytest

import kv4_ref as ref
import sib200

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HEADS = {(14, 2, 64), (12, 2, 128), (28, 4, 128), (64, 8, 128), (4, 4, 128), (1, 1, 64)}


def dims_of(hq, hkv, D):
    return dict(hidden=hq * D, n_q_heads=hq, n_kv_heads=hkv, head_dim=D, intermediate=0,
                rope_theta=1e6, rms_eps=1e-6)


def up(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Cache:
    """A KV4 with shuffled pages and the 64-bit values of what was appended."""

    def __init__(self, ctx, heads, n_seqs, max_ctx, page_len, seed=0, spare=5):
        self.ctx, (self.hq, self.hkv, self.D) = ctx, heads
        self.dims = dims_of(*heads)
        self.P = page_len
        per = -(-max_ctx // page_len)
        self.n_pages = n_seqs * per + spare
        self.kv = ctx.kv4(self.dims, n_seqs, max_ctx, self.n_pages, page_len)
        self.rng = np.random.default_rng(seed)
        self.k = [np.zeros((max_ctx, self.hkv, self.D)) for _ in range(n_seqs)]
        self.v = [np.zeros((max_ctx, self.hkv, self.D)) for _ in range(n_seqs)]

    def shuffle(self, lens):
        ids = self.rng.permutation(self.n_pages)
        need = [-(-n // self.P) for n in lens]
        seqs = [s for s, n in enumerate(need) if n]
        self.kv.assign(seqs, [need[s] for s in seqs], ids[:sum(need)])

    def append(self, runs, k, v):
        kd, vd = up(k.astype(np.float32)), up(v.astype(np.float32))
        torch.cuda.synchronize()
        self.kv.append(kd, vd, runs)
        self.ctx.sync()
        kq, vq = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
        at = 0
        for s, p, c in runs:
            self.k[s][p:p + c], self.v[s][p:p + c] = kq[at:at + c], vq[at:at + c]
            at += c

    def random(self, runs, kscale=1.0, vscale=1.0):
        T = sum(c for _, _, c in runs)
        shape = (T, self.hkv, self.D)
        self.append(runs, self.rng.standard_normal(shape) * kscale,
                    self.rng.standard_normal(shape) * vscale)

    def attend(self, q, runs):
        qd = up(q.astype(np.float32))
        out = torch.full(q.shape, 7.0, device="cuda")
        torch.cuda.synchronize()
        self.ctx.attention_kv4(self.kv, self.dims, qd, runs, out)
        self.ctx.status()
        return out.cpu().numpy()

    def check(self, got, q, runs, chain=None, every=1):
        """Every row within its bound; the whole within 2^-17 (an operand kept to
        11 bits instead of 22 would put it at 2^-12) plus what fp32 scores of that
        size cost: the product with log2(e) / sqrt(D) and the difference to the
        maximum round a score s twice, 2^-24 |s| each, in the exponent of the
        numerator and of the denominator: 2^-22 |s| together.  every: of a run's
        tokens the first, each every-th and the last."""
        at, num, den, top = 0, 0.0, 0.0, 0.0
        for s, p, c in runs:
            for j in range(c):
                if j % every and j != c - 1:
                    at += 1
                    continue
                n = p + j + 1
                k, v = self.k[s][:n], self.v[s][:n]
                want, bound, t = ref.attention(q[at].astype(np.float32), k, v)
                top = max(top, t)
                steps = chain or 4 + n / 16
                bound = bound + ref.steps_bound(v, n, steps) + 1e-30
                err = np.abs(got[at] - want)
                assert np.all(err <= bound), (s, n, (err / bound).max())
                num += (err ** 2).sum()
                den += (want ** 2).sum()
                at += 1
        norm = 2.0 ** -17 + 2.0 ** -22 * top
        assert num <= (norm ** 2) * den, np.sqrt(num / den)


# ---------------------------------------------------------------- writing --
@pytest.mark.parametrize("heads,page", [((14, 2, 64), 16), ((12, 2, 128), 48), ((28, 4, 128), 64)])
def test_append_writes_the_rule_and_the_layout(si_ctx, heads, page):
    c = Cache(si_ctx, heads, 5, 200, page, seed=1)
    hq, hkv, D = heads
    c.shuffle([200, 0, 37, 1, 100])
    runs = [(0, 0, 130), (2, 3, 30), (0, 130, 1), (1, 0, 17), (4, 99, 1), (3, 0, 1), (2, 0, 0)]
    T = sum(r[2] for r in runs)
    k = c.rng.standard_normal((T, hkv, D)).astype(np.float32)
    v = (c.rng.standard_normal((T, hkv, D)) * np.exp(c.rng.standard_normal((T, 1, 1)) * 6)).astype(np.float32)
    # ties of either sign, zeros, the smallest and the largest values
    k[0, 0, :32] = 1.0
    k[0, 0, 7] = -1.0
    k[1, 0, :32] = -1.0
    k[1, 0, 31] = 1.0
    k[2] = 0.0
    k[3, 0, :] = 1e-45
    k[4, 0, :] = np.linspace(-520000, 520000, D)
    k[5, 0, :] = np.linspace(1e-9, 1e-6, D)
    before = np.zeros((c.n_pages, hkv, page // 16, ref.group_bytes(D)), np.uint8)
    c.append(runs, k, v)
    si_ctx.status()
    n = before.size

    class W:
        __cuda_array_interface__ = {"data": (c.kv.device_ptr(0), False), "shape": (n,), "typestr": "|u1",
                                    "version": 3, "strides": None}
    pool = torch.as_tensor(W(), device="cuda").cpu().numpy().reshape(before.shape)
    (kc, ks), (vc, vs) = ref.quantise(k), ref.quantise(v)
    at = 0
    for s, p, cnt in runs:
        pages = c.kv.pages(s)
        for j in range(cnt):
            for h in range(hkv):
                for is_v, cc, ss in ((False, kc, ks), (True, vc, vs)):
                    ref.place(before, pages[(p + j) // page], h, (p + j) % page, is_v, D, page,
                              cc[at, h], ss[at, h])
            at += 1
    np.testing.assert_array_equal(pool, before)  # and nothing else was written
    # read back, in another order of runs
    back = [(4, 99, 1), (0, 5, 100), (2, 3, 30)]
    T2 = sum(r[2] for r in back)
    ko, vo = (torch.full((T2, hkv, D), 9.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read(back, ko, vo)
    si_ctx.status()
    want_k = np.concatenate([c.k[s][p:p + n] for s, p, n in back])
    want_v = np.concatenate([c.v[s][p:p + n] for s, p, n in back])
    np.testing.assert_array_equal(ko.cpu().numpy(), want_k.astype(np.float32))
    np.testing.assert_array_equal(vo.cpu().numpy(), want_v.astype(np.float32))
    ko.fill_(3.0)
    torch.cuda.synchronize()
    c.kv.read(back, None, vo)
    si_ctx.status()
    assert torch.all(ko == 3.0)
    c.kv.free()


@pytest.mark.parametrize("heads", [(8, 1, 64), (9, 3, 64), (5, 5, 128), (64, 8, 128)])
def test_ties_infinities_and_nan_of_every_row(si_ctx, heads):
    """The first of a block's values of largest magnitude gives the sign of its scale,
    whichever lane holds it; a block with a NaN reads as NaN, one with an infinity
    as infinities and NaN."""
    c = Cache(si_ctx, heads, 1, 64, 16, seed=12)
    hq, hkv, D = heads
    c.shuffle([64])
    k = c.rng.choice([-1.0, 1.0, 0.25, -0.25], (64, hkv, D)).astype(np.float32)
    v = c.rng.choice([-2.0, 2.0], (64, hkv, D)).astype(np.float32)
    k[40:44, :, 5] = np.inf
    k[42:44, :, 37] = -np.inf
    v[50, :, D - 1] = np.nan
    c.append([(0, 0, 64)], k, v)
    gk, gv = (torch.empty((64, hkv, D), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read([(0, 0, 64)], gk, gv)
    si_ctx.status()
    for got, rows in ((gk, k), (gv, v)):
        with np.errstate(invalid="ignore"):
            want = ref.values(*ref.quantise(rows)).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def test_rows_that_are_not_16_byte_aligned(si_ctx):
    c = Cache(si_ctx, (14, 2, 64), 1, 40, 16, seed=21)
    k = c.rng.standard_normal((33, 2, 64)).astype(np.float32)
    v = c.rng.standard_normal((33, 2, 64)).astype(np.float32)
    buf = torch.zeros(2, 33 * 128 + 1, device="cuda")
    buf[0, 1:], buf[1, :-1] = up(k).view(-1), up(v).view(-1)
    torch.cuda.synchronize()
    c.kv.append(buf[0, 1:], buf[1], [(0, 0, 33)])
    ko, vo = (torch.zeros(33, 2, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read([(0, 0, 33)], ko, vo)
    si_ctx.status()
    for x, y in ((k, ko), (v, vo)):
        np.testing.assert_array_equal(y.cpu().numpy(), ref.values(*ref.quantise(x)).astype(np.float32))
    c.kv.free()


def test_append_of_many_runs(si_ctx):
    """More runs than one launch takes, one token each."""
    c = Cache(si_ctx, (1, 1, 64), 700, 3, 16, seed=2)
    runs = [(s, s % 3, 1) for s in range(700)]
    c.random(runs)
    ko, vo = (torch.zeros(700, 1, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read(runs, ko, vo)
    si_ctx.status()
    want = np.stack([c.k[s][s % 3] for s in range(700)]).astype(np.float32)
    np.testing.assert_array_equal(ko.cpu().numpy(), want)
    q = c.rng.standard_normal((700, 1, 64))
    zero = [(s, 0, 1) for s in range(0, 700, 3)]  # their only written position
    got = c.attend(q[:len(zero)], zero)
    c.check(got, q, zero)
    c.kv.free()


# -------------------------------------------------------------- attention --
@pytest.mark.parametrize("heads", sorted(HEADS))
@pytest.mark.parametrize("page", [16, 48, 128])
def test_decode_attention_ragged(si_ctx, heads, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 600, 1025]
    c = Cache(si_ctx, heads, len(lens), 1100, page, seed=3)
    c.shuffle(lens)
    c.random([(s, 0, n) for s, n in enumerate(lens)])
    runs = [(s, n - 1, 1) for s, n in enumerate(lens)] + [(11, -1, 1), (12, 500, 1), (12, 1024, 1)]
    q = c.rng.standard_normal((len(runs), heads[0], heads[2]))
    got = c.attend(q, runs)
    assert np.all(got[len(lens)] == 0)  # no keys
    c.check(got, q, runs)
    c.kv.free()


def test_decode_attention_long_context(si_ctx):
    c = Cache(si_ctx, (8, 1, 128), 2, 40000, 64, seed=4)
    c.random([(0, 0, 40000), (1, 0, 77)])
    runs = [(0, 39998, 1), (1, 76, 1)]
    q = c.rng.standard_normal((2, 8, 128))
    c.check(c.attend(q, runs), q, runs)
    c.kv.free()


@pytest.mark.parametrize("kscale,vscale,qscale", [(1e-4, 1.0, 1e4), (1e3, 1.0, 1e-3),
                                                  (1.0, 1e-5, 1.0), (1.0, 3e4, 1.0),
                                                  (1e3, 1e-3, 1e-30), (1e-3, 1.0, 1e6)])
@pytest.mark.parametrize("total,count", [(300, 1), (300, 40), (2700, 131)])
def test_attention_keeps_its_bits_at_any_scale(si_ctx, kscale, vscale, qscale, total, count):
    c = Cache(si_ctx, (12, 2, 128), 1, total, 64, seed=5)
    c.random([(0, 0, total)], kscale, vscale)
    runs = [(0, total - count, count)]
    q = c.rng.standard_normal((count, 12, 128)) * qscale
    c.check(c.attend(q, runs), q, runs, every=13)
    c.kv.free()


def test_scales_that_grow_along_the_keys(si_ctx):
    """Values whose size rises by 2^24 along the sequence, and one head of large ones."""
    c = Cache(si_ctx, (14, 2, 64), 1, 520, 16, seed=6)
    k = c.rng.standard_normal((520, 2, 64))
    v = c.rng.standard_normal((520, 2, 64)) * 2.0 ** np.linspace(-12, 12, 520)[:, None, None]
    c.append([(0, 0, 520)], k, v)
    q = c.rng.standard_normal((2, 14, 64))
    runs = [(0, 519, 1), (0, 250, 1)]
    c.check(c.attend(q, runs), q, runs)
    v = v[::-1].copy()
    c.append([(0, 0, 520)], k, v)
    c.check(c.attend(q, runs), q, runs)
    c.kv.free()


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("n,count", [(131, 1), (131, 3), (131, 20), (3331, 131)])
def test_what_lies_behind_a_sequence_is_not_seen(si_ctx, heads, n, count):
    """Rows past the last position hold NaN and infinite scales."""
    c = Cache(si_ctx, heads, 1, n + 125, 64, seed=7)
    hq, hkv, D = heads
    c.random([(0, 0, n)])
    bad = np.full((125, hkv, D), np.inf)
    bad[::2] = np.nan
    kd, vd = up(bad.astype(np.float32)), up(bad.astype(np.float32))
    torch.cuda.synchronize()
    c.kv.append(kd, vd, [(0, n, 125)])
    runs = [(0, n - count, count)]
    q = c.rng.standard_normal((count, hq, D))
    got = c.attend(q, runs)
    assert np.all(np.isfinite(got))
    c.check(got, q, runs, every=13)
    # and a NaN inside shows
    if count < 100:
        assert np.isnan(c.attend(q, [(0, n + 3, count)])).all()
    c.kv.free()


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("prefix,where", [(20, 0), (20, 40), (20, 99), (4100, 0), (4100, 57)])
def test_a_nan_inside_a_prompt_reaches_only_later_rows(si_ctx, heads, prefix, where):
    """Position prefix + where of a prompt holds a NaN value: the queries before it do
    not see it."""
    c = Cache(si_ctx, heads, 1, prefix + 100, 32, seed=13)
    hq, hkv, D = heads
    c.random([(0, 0, prefix + 100)])
    bad = np.full((1, hkv, D), np.nan, np.float32)
    one = np.ones((1, hkv, D), np.float32)
    kd, vd = up(one), up(bad)
    torch.cuda.synchronize()
    c.kv.append(kd, vd, [(0, prefix + where, 1)])
    q = c.rng.standard_normal((100, hq, D))
    got = c.attend(q, [(0, prefix, 100)])
    if where:
        c.check(got[:where], q[:where], [(0, prefix, where)], every=7)
    assert np.isnan(got[where:]).all()
    c.kv.free()


def test_sharp_and_flat_softmax(si_ctx):
    c = Cache(si_ctx, (28, 4, 128), 1, 700, 64, seed=8)
    c.random([(0, 0, 700)])
    for qs in (0.0, 1e-3, 30.0):
        q = c.rng.standard_normal((2, 28, 128)) * qs
        runs = [(0, 699, 1), (0, 330, 1)]
        c.check(c.attend(q, runs), q, runs)
    c.kv.free()


# Runs that the prompt kernel takes: from an empty cache, from odd prefixes, with
# few tokens (the key axis split over CTAs) and a ragged last tile of rows and keys.
PROMPTS = [((28, 4, 128), 0, 530), ((64, 8, 128), 520, 131), ((12, 2, 128), 2500, 131),
           ((14, 2, 64), 3200, 131), ((64, 8, 128), 7990, 17), ((4, 4, 128), 9000, 24),
           ((8, 1, 128), 6001, 129), ((6, 2, 128), 4001, 71)]


@pytest.mark.parametrize("heads,prefix,count", PROMPTS)
@pytest.mark.parametrize("exact", [False, True])
def test_prompt_attention(si_ctx, heads, exact, prefix, count):
    c = Cache(si_ctx, heads, 2, prefix + count + 9, 48, seed=9)
    c.shuffle([0, prefix + count])
    c.random([(1, 0, prefix + count)])
    runs = [(1, prefix, count)]
    q = c.rng.standard_normal((count, heads[0], heads[2]))
    si_ctx.set_exact_attention(exact)
    try:
        got = c.attend(q, runs)
    finally:
        si_ctx.set_exact_attention(False)
    c.check(got, q, runs, every=11)
    c.kv.free()


@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64), (64, 8, 128)])
@pytest.mark.parametrize("prefix,count", [(0, 16), (0, 150), (37, 131), (500, 17)])
def test_short_prompt_attention(si_ctx, heads, prefix, count):
    """Runs with too little work for the prompt kernel."""
    c = Cache(si_ctx, heads, 2, prefix + count + 9, 48, seed=9)
    c.shuffle([0, prefix + count])
    c.random([(1, 0, prefix + count)])
    runs = [(1, prefix, count)]
    q = c.rng.standard_normal((count, heads[0], heads[2]))
    c.check(c.attend(q, runs), q, runs, every=5)
    c.kv.free()


def test_mixed_batch_of_prompts_and_tokens(si_ctx):
    """Prompts between single tokens, proposals and padding, in one call; rows outside
    the call's stay."""
    c = Cache(si_ctx, (12, 2, 128), 6, 3000, 32, seed=10)
    lens = [300, 2999, 40, 64, 65, 10]
    c.random([(s, 0, n) for s, n in enumerate(lens)])
    runs = [(0, 299, 1), (1, 2880, 119), (2, 35, 5), (5, -1, 2), (3, 0, 64), (4, 64, 1), (0, 0, 0),
            (1, 2700, 150)]
    T = sum(r[2] for r in runs)
    q = c.rng.standard_normal((T, 12, 128))
    qd, out = up(q.astype(np.float32)), torch.full((T + 2, 12, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    si_ctx.attention_kv4(c.kv, c.dims, qd, runs, out[1:])
    si_ctx.status()
    got = out.cpu().numpy()
    assert np.all(got[0] == 7.0) and np.all(got[-1] == 7.0)
    c.check(got[1:-1], q, runs, every=9)
    # the same call again gives the same bits
    again = torch.zeros_like(out)
    torch.cuda.synchronize()
    si_ctx.attention_kv4(c.kv, c.dims, qd, runs, again[1:])
    si_ctx.status()
    np.testing.assert_array_equal(again.cpu().numpy()[1:-1], got[1:-1])
    c.kv.free()


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64), (3, 3, 128)])
def test_many_prompts_in_one_call(si_ctx, heads):
    """More prompts than one launch takes, of odd lengths, several of one sequence,
    between single tokens; a NaN in one sequence stays in its own rows."""
    c = Cache(si_ctx, heads, 12, 1000, 48, seed=26)
    lens = [900, 64, 333, 1000, 17, 640, 512, 129, 777, 48, 801, 96]
    c.shuffle(lens)
    c.random([(s, 0, n) for s, n in enumerate(lens)])
    bad = np.full((1, heads[1], heads[2]), np.nan, np.float32)
    c.append([(6, 0, 1)], bad, bad)
    runs = []
    for s, n in enumerate(lens):
        for count in (16 + 7 * s, 16 + s, 1):
            if count <= n:
                runs.append((s, n - count, count))
    runs += [(3, 500, 131), (0, 0, 64), (0, 0, 16), (8, 700, 13), (10, 5, 14), (8, 600, 12)]
    assert sum(r[2] >= 16 for r in runs) > 16
    q = c.rng.standard_normal((sum(r[2] for r in runs), heads[0], heads[2]))
    got = c.attend(q, runs)
    at, good = 0, np.ones(len(q), bool)
    for s, p, count in runs:
        good[at:at + count] = s != 6
        at += count
    assert np.isnan(got[~good]).all()
    c.check(got[good], q[good], [r for r in runs if r[0] != 6], every=11)
    c.kv.free()


def test_prompts_with_too_many_keys_for_one_launch(si_ctx):
    """Operands of three prompts that would take a gigabyte together."""
    c = Cache(si_ctx, (8, 8, 128), 1, 40000, 128, seed=27)
    c.random([(0, 0, 40000)])
    runs = [(0, 33000, 16), (0, 39980, 20), (0, 100, 40), (0, 36000, 17)]
    q = c.rng.standard_normal((sum(r[2] for r in runs), 8, 128))
    c.check(c.attend(q, runs), q, runs, every=50)
    c.kv.free()


# ------------------------------------------------------------------- pages --
def test_fork_write_and_compact(si_ctx):
    c = Cache(si_ctx, (12, 2, 128), 4, 200, 32, seed=11, spare=10)
    c.kv.assign([3], [2], [17, 30])  # someone else's pages
    c.kv.release([3])
    c.random([(0, 0, 150)])
    c.kv.fork([0, 0], [1, 2], [150, 70])
    for s, n in ((1, 150), (2, 70)):
        c.k[s][:n], c.v[s][:n] = c.k[0][:n], c.v[0][:n]
    assert c.kv.pages(1)[:4] == c.kv.pages(0)[:4] and c.kv.pages(1)[4] != c.kv.pages(0)[4]
    q = c.rng.standard_normal((3, 12, 128))
    runs = [(0, 149, 1), (1, 149, 1), (2, 69, 1)]
    got = c.attend(q, runs)
    c.check(got, q, runs)
    c.random([(1, 150, 20), (2, 10, 5), (0, 150, 1)])  # 2 writes into a shared page
    runs = [(0, 150, 1), (1, 169, 1), (2, 69, 1)]
    c.check(c.attend(q, runs), q, runs)
    c.kv.release([0], [100])
    c.kv.release([2])
    runs = [(0, 99, 1), (1, 169, 1)]
    before = c.attend(q[:2], runs)
    used = c.kv.compact()
    assert used == c.n_pages - c.kv.free_pages()
    assert all(p < used for s in range(4) for p in c.kv.pages(s))
    np.testing.assert_array_equal(c.attend(q[:2], runs), before)
    c.kv.free()


def test_large_page_changes(si_ctx):
    """More table entries, counts and copies than one launch takes."""
    n = 5000
    c = Cache(si_ctx, (1, 1, 64), 3, n * 16, 16, seed=12, spare=0)
    ids = np.concatenate([np.arange(1, 3 * n, 2)[:n], ])
    c.kv.assign([1], [n], ids)
    T = 64
    c.random([(1, 16 * i, 1) for i in range(0, n, n // T)][:T])
    spots = [(1, 16 * i, 1) for i in range(0, n, n // T)][:T]
    assert c.kv.compact() == n
    ko, vo = (torch.zeros(T, 1, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read(spots, ko, vo)
    si_ctx.status()
    want = np.stack([c.v[1][p] for _, p, _ in spots]).astype(np.float32)
    np.testing.assert_array_equal(vo.cpu().numpy(), want)
    c.kv.fork([1], [2], [n * 16])
    assert c.kv.pages(2) == c.kv.pages(1) and c.kv.free_pages() == 2 * n
    c.kv.read([(2, p, k) for _, p, k in spots], ko, vo)
    si_ctx.status()
    np.testing.assert_array_equal(vo.cpu().numpy(), want)
    c.kv.free()


def test_pool_beyond_four_gigabytes(si_ctx):
    """Pages at the end of a pool of 5.9 GB: written, read, attended by both kernels,
    copied and moved."""
    heads, P = (64, 8, 128), 128
    dims = dims_of(*heads)
    n_pages = 40000
    assert n_pages * sib200.kv4_page_bytes(dims, P) > 5 << 30
    c = Cache.__new__(Cache)
    c.ctx, (c.hq, c.hkv, c.D), c.dims, c.P, c.n_pages = si_ctx, heads, dims, P, n_pages
    c.kv = si_ctx.kv4(dims, 2, 1024, n_pages, P)
    c.rng = np.random.default_rng(22)
    c.k = [np.zeros((1024, 8, 128)) for _ in range(2)]
    c.v = [np.zeros((1024, 8, 128)) for _ in range(2)]
    c.kv.assign([0], [8], np.arange(n_pages - 8, n_pages)[::-1])
    c.random([(0, 0, 1000)])
    runs = [(0, 999, 1), (0, 868, 131)]
    q = c.rng.standard_normal((132, 64, 128))
    got = c.attend(q, runs)
    c.check(got, q, runs, every=40)
    c.kv.fork([0], [1], [1000])        # the last page is copied to the front
    c.k[1], c.v[1] = c.k[0], c.v[0]
    one = [(1, 999, 1)]
    first = c.attend(q[:1], one)
    c.check(first, q[:1], one)
    assert c.kv.compact() == 9
    np.testing.assert_array_equal(c.attend(q[:1], one), first)
    ko, vo = (torch.zeros(1000, 8, 128, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.kv.read([(0, 0, 1000)], ko, vo)
    si_ctx.status()
    np.testing.assert_array_equal(vo.cpu().numpy(), c.v[0][:1000].astype(np.float32))
    c.kv.free()


def test_workspaces_after_a_capture():
    """A workspace that a graph holds outlives its growth; those that came after the
    capture do not pile up."""
    def filled(ctx):
        c = Cache(ctx, (12, 2, 128), 1, 2048, 64, seed=24)
        c.random([(0, 0, 2048)])
        return c, torch.randn(2048, 12, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(6))

    def attend(c, q, count, out):
        c.ctx.attention_kv4(c.kv, c.dims, q[:count], [(0, 2048 - count, count)], out)

    counts = range(300, 2049, 76)
    ctx = sib200.Context(0, max_positions=64, head_dim=128)
    c, q = filled(ctx)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    for count in counts:  # not all need less than the last: fewer rows split the keys
        attend(c, q, count, out)
    ctx.status()
    need = ctx.scratch_bytes()
    c.kv.free()
    ctx.close()

    ctx = sib200.Context(0, max_positions=64, head_dim=128)
    c, q = filled(ctx)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    attend(c, q, 200, out)
    ctx.status()
    want = out.clone()
    torch.cuda.synchronize()
    first = ctx.scratch_bytes()
    graph = ctx.capture(lambda: attend(c, q, 200, out))
    for count in counts:
        attend(c, q, count, out)
    ctx.status()
    assert ctx.scratch_bytes() <= first + need
    out.zero_()
    torch.cuda.synchronize()
    graph.launch()
    ctx.status()
    assert torch.equal(out, want)
    graph.free()
    c.kv.free()
    ctx.close()


def test_captured_calls_share_the_workspace(si_ctx):
    """Two graphs of append and attention calls (tokens, and a prompt with tokens) over
    the same workspaces, replayed in turn with new inputs, against eager calls."""
    c = Cache(si_ctx, (12, 2, 128), 3, 3000, 64, seed=23)
    lens = [2700, 900, 64]
    c.random([(s, 0, n) for s, n in enumerate(lens)])
    runs_a = [(0, 2699, 1), (1, 899, 1), (2, -1, 1)]
    runs_b = [(0, 2560, 140), (1, 880, 20)]
    qa, qb = torch.zeros(3, 12, 128, device="cuda"), torch.zeros(160, 12, 128, device="cuda")
    new = torch.zeros(2, 2, 2, 128, device="cuda")
    oa, ob = torch.zeros_like(qa), torch.zeros_like(qb)
    torch.cuda.synchronize()

    def call_a():
        c.kv.append(new[0], new[1], [(0, 2699, 1), (1, 899, 1)])
        si_ctx.attention_kv4(c.kv, c.dims, qa, runs_a, oa)

    def call_b():
        si_ctx.attention_kv4(c.kv, c.dims, qb, runs_b, ob)

    call_a()
    call_b()
    ga, gb = si_ctx.capture(call_a), si_ctx.capture(call_b)
    g = torch.Generator("cuda").manual_seed(5)
    for _ in range(3):
        for t in (qa, qb, new):
            t.normal_(generator=g)
        torch.cuda.synchronize()
        ga.launch()
        gb.launch()
        ga.launch()
        si_ctx.status()
        a, b = oa.clone(), ob.clone()
        oa.zero_()
        ob.zero_()
        torch.cuda.synchronize()
        call_a()
        call_b()
        si_ctx.status()
        assert torch.equal(a, oa) and torch.equal(b, ob)
        kq = ref.values(*ref.quantise(new[0].cpu().numpy()))
        vq = ref.values(*ref.quantise(new[1].cpu().numpy()))
        for i, (s, p) in enumerate(((0, 2699), (1, 899))):
            c.k[s][p], c.v[s][p] = kq[i], vq[i]
        c.check(a.cpu().numpy(), qa.cpu().numpy(), runs_a)
        c.check(b.cpu().numpy(), qb.cpu().numpy(), runs_b, every=39)
    ga.free()
    gb.free()
    c.kv.free()


# ------------------------------------------------------------- layer steps --
DIMS = dict(hidden=896, n_q_heads=14, n_kv_heads=2, head_dim=64, intermediate=4864,
            rope_theta=1e6, rms_eps=1e-6)
DIMS128 = dict(hidden=1536, n_q_heads=12, n_kv_heads=2, head_dim=128, intermediate=8960,
               rope_theta=1e6, rms_eps=1e-6)


def expected_attn_step(ctx, layer, dims, x, kv, runs):
    """run_layer's function with the cache's values: the library's own projections,
    the reference's rope on the host, attention in 64 bits; (y, cache rows)."""
    H, D, hq, hkv = dims["hidden"], dims["head_dim"], dims["n_q_heads"], dims["n_kv_heads"]
    QD, KVD = hq * D, hkv * D
    T = x.shape[0]
    host = layer.host()
    qs, d = torch.zeros(T, H, dtype=torch.int8, device="cuda"), torch.zeros(T, H // 32, dtype=torch.int16, device="cuda")
    bias, qkv = up(np.concatenate([host["bq"], host["bk"], host["bv"]])), torch.zeros(T, QD + 2 * KVD, device="cuda")
    norm = up(host["norm"])
    torch.cuda.synchronize()
    ctx.rmsnorm_q8(x, norm, T, H, dims["rms_eps"], None, qs, d)
    ctx.matmul(layer.matrix(0), qs, d, T, bias, qkv)
    ctx.sync()
    p = qkv.cpu().numpy()
    q, k, v = p[:, :QD].copy(), p[:, QD:QD + KVD].copy(), p[:, QD + KVD:].reshape(T, hkv, D)
    at = 0
    for s, pos, c in runs:
        for j in range(c):
            for a, n in ((q[at], hq), (k[at], hkv)):
                ctx.L.si_ref_rope(sib200._p(a), n, pos + j, D, dims["rope_theta"])
            at += 1
    k = k.reshape(T, hkv, D)
    kq, vq = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
    at = 0
    attn = np.zeros((T, QD))
    for s, pos, c in runs:
        kv[s][0][pos:pos + c], kv[s][1][pos:pos + c] = kq[at:at + c], vq[at:at + c]
        for j in range(c):
            n = pos + j + 1
            attn[at + j] = ref.attention(q[at + j].reshape(hq, D), kv[s][0][:n], kv[s][1][:n])[0].reshape(-1)
        at += c
    a = up(attn.astype(np.float32))
    aq, ad = torch.zeros(T, QD, dtype=torch.int8, device="cuda"), torch.zeros(T, QD // 32, dtype=torch.int16, device="cuda")
    y = torch.zeros(T, H, device="cuda")
    torch.cuda.synchronize()
    ctx.q8_quantize(a, T, QD, aq, ad)
    ctx.matmul(layer.matrix(1), aq, ad, T, None, y)
    ctx.sync()
    return y.cpu().numpy()


@pytest.mark.parametrize("dims", [DIMS, DIMS128])
def test_layer_steps(dims):
    """A prompt, then a mixed step, then decode steps: outputs against the composed
    expectation, the cache's rows bit for bit."""
    ctx = sib200.Context(0, max_positions=512, rope_theta=1e6, head_dim=dims["head_dim"])
    layer = ctx.layer_synth(dims, 5)
    D, hkv, H = dims["head_dim"], dims["n_kv_heads"], dims["hidden"]
    kv = ctx.kv4(dims, 3, 512, 40, 32)
    want_kv = [(np.zeros((512, hkv, D)), np.zeros((512, hkv, D))) for _ in range(3)]
    g = torch.Generator("cuda").manual_seed(3)
    for runs in ([(0, 0, 50)], [(0, 50, 1), (2, 0, 33), (1, 0, 3)], [(0, 51, 1), (1, 3, 1), (2, 33, 1)]):
        T = sum(r[2] for r in runs)
        x, y = torch.randn(T, H, device="cuda", generator=g), torch.zeros(T, H, device="cuda")
        torch.cuda.synchronize()
        layer.step_dev(kv, x, runs, y)
        ctx.status()
        want = expected_attn_step(ctx, layer, dims, x, want_kv, runs)
        got = y.cpu().numpy()
        # one flipped Q8 code of the attention output moves a row by about
        # 1 / 127 of one input's share: the layer bar of the other step tests
        for t in range(T):
            e = np.linalg.norm(got[t] - want[t]) / np.linalg.norm(want[t])
            assert e < 1e-2, (runs, t, e)
        rows = torch.zeros(2, T, hkv, D, device="cuda")
        torch.cuda.synchronize()
        kv.read(runs, rows[0], rows[1])
        ctx.status()
        for i in (0, 1):
            w = np.concatenate([want_kv[s][i][p:p + c] for s, p, c in runs]).astype(np.float32)
            np.testing.assert_array_equal(rows[i].cpu().numpy(), w)
    # the whole layer: y = h + mlp runs and differs from the attention alone
    z = torch.zeros_like(y)
    torch.cuda.synchronize()
    layer.step_dev(kv, x, runs, z, sib200.SI_LAYER_FULL)
    ctx.status()
    assert torch.isfinite(z).all() and not torch.equal(z, y)
    kv.free()
    layer.free()
    ctx.close()


def test_captured_steps_equal_eager_ones():
    """A two-layer step with device lengths, captured once and replayed, against
    steps with host runs, over a page border; a later larger call does not
    disturb the graph."""
    dims = DIMS128
    ctx = sib200.Context(0, max_positions=512, rope_theta=1e6, head_dim=128)
    layers = [ctx.layer_synth(dims, 20 + i) for i in range(2)]
    B, H, L = 3, dims["hidden"], 512
    lens = [30, 97, 64]
    g = torch.Generator("cuda").manual_seed(4)
    x0 = torch.randn(B, H, device="cuda", generator=g)
    prompt = torch.randn(sum(lens), H, device="cuda", generator=g)
    tmp = torch.zeros_like(prompt)

    def caches():
        kvs = [ctx.kv4(dims, B, L, 60, 32) for _ in layers]
        for kv, layer in zip(kvs, layers):
            layer.step_dev(kv, prompt, [(s, 0, n) for s, n in enumerate(lens)], tmp)
        return kvs

    torch.cuda.synchronize()
    ka, kb = caches(), caches()
    xa, xb = [x0.clone(), torch.zeros_like(x0)], [x0.clone(), torch.zeros_like(x0)]
    st = ctx.decode_state([n + 1 for n in lens], L)
    for kv in kb:
        kv.reserve([(s, n, 10) for s, n in enumerate(lens)])
    torch.cuda.synchronize()

    def step():
        for j, (layer, kv) in enumerate(zip(layers, kb)):
            layer.decode_state_dev(kv, xb[j % 2], st, xb[(j + 1) % 2], sib200.SI_LAYER_FULL)
        st.advance()

    def eager(i):
        for j, (layer, kv) in enumerate(zip(layers, ka)):
            layer.step_dev(kv, xa[j % 2], [(s, n + i, 1) for s, n in enumerate(lens)],
                           xa[(j + 1) % 2], sib200.SI_LAYER_FULL)

    step()
    eager(0)
    graph = ctx.capture(step)
    for i in range(1, 6):
        if i == 3:  # grows the context's buffers
            big = torch.randn(400, H, device="cuda", generator=g)
            torch.cuda.synchronize()
            other = ctx.kv4(dims, 1, 512, 20, 32)
            layers[0].step_dev(other, big, [(0, 0, 400)], torch.zeros_like(big), sib200.SI_LAYER_FULL)
            ctx.sync()
            other.free()
        graph.launch()
        eager(i)
        ctx.status()
        a, b = xa[0].cpu().numpy(), xb[0].cpu().numpy()
        # the split of the keys differs, so a Q8 code may flip on the way
        assert np.linalg.norm(a - b) <= 1e-2 * np.linalg.norm(a), i
    rows = [(s, 0, n + 1) for s, n in enumerate(lens)]
    T = sum(r[2] for r in rows)
    out = torch.zeros(4, T, 2, 128, device="cuda")
    torch.cuda.synchronize()
    ka[0].read(rows, out[0], out[1])
    kb[0].read(rows, out[2], out[3])
    ctx.status()
    assert torch.equal(out[:2], out[2:])
    # changes of the pages are refused while a graph is captured
    with pytest.raises(sib200.SiError):
        ctx.capture(lambda: kb[0].fork([0], [1], [3]))
    with pytest.raises(sib200.SiError):
        ctx.capture(lambda: layers[0].step_dev(ka[0], x0, [(s, 300, 1) for s in range(B)], xb[1]))
    graph.free()
    ctx.close()


def test_device_length_steps_refuse_pages_that_are_not_theirs():
    ctx = sib200.Context(0, max_positions=128, rope_theta=1e6, head_dim=64)
    layer = ctx.layer_synth(DIMS, 6)
    kv = ctx.kv4(DIMS, 2, 128, 12, 16)
    x, y = torch.randn(2, 896, device="cuda"), torch.zeros(2, 896, device="cuda")
    p = torch.randn(16, 896, device="cuda")
    z = torch.zeros_like(p)
    torch.cuda.synchronize()
    layer.step_dev(kv, p, [(0, 0, 16)], z)
    kv.fork([0], [1], [16])
    ctx.status()
    want = torch.zeros(2, 16, 2, 64, device="cuda")
    got = torch.zeros_like(want)
    torch.cuda.synchronize()
    kv.read([(0, 0, 16)], want[0], want[1])
    st = ctx.decode_state([16, 16], 128)   # both would write position 15 of a shared page
    layer.decode_state_dev(kv, x, st, y)
    with pytest.raises(sib200.SiError) as e:
        ctx.status()
    assert e.value.status == sib200.SI_ERR_INVALID
    kv.read([(1, 0, 16)], got[0], got[1])
    ctx.status()
    assert torch.equal(got, want)
    st.set([17, 17])                       # no page there
    layer.decode_state_dev(kv, x, st, y)
    with pytest.raises(sib200.SiError):
        ctx.status()
    kv.reserve([(0, 16, 1), (1, 16, 1)])
    layer.decode_state_dev(kv, x, st, y)
    ctx.status()
    ctx.close()


# --------------------------------------------------------------- refusals --
def test_refusals(si_ctx):
    dims = dims_of(12, 2, 128)
    t = torch.zeros(64, 12, 128, device="cuda")
    bad = sib200.SiError

    def no(f, *a, **k):
        with pytest.raises(bad) as e:
            f(*a, **k)
        assert e.value.status == sib200.SI_ERR_INVALID, str(e.value)

    for page in (0, 8, 24, -16, 8192):
        no(si_ctx.kv4, dims, 1, 64, 4, page)
    for a in ((0, 64, 4), (1, 0, 4), (1, 64, 0), (1 << 20, 1 << 30, 4), (1, 64, 1 << 30)):
        no(si_ctx.kv4, dims, *a, 16)
    no(si_ctx.kv4, dict(dims, head_dim=96), 1, 64, 4, 16)
    pool = torch.zeros(4 * sib200.kv4_page_bytes(dims, 16) + 8, dtype=torch.uint8, device="cuda")
    no(si_ctx.kv4, dims, 1, 64, 4, 16, pool[8:])
    with pytest.raises(ValueError):
        si_ctx.kv4(dims, 1, 64, 5, 16, pool)
    kv = si_ctx.kv4(dims, 2, 60, 4, 16, pool)
    kv.append(t, t, [(0, 0, 20)])
    free = kv.free_pages()
    no(kv.append, t, t, [(0, 19, 1), (0, 18, 2)])       # one position twice
    no(kv.append, t, t, [(0, 60, 1)])                   # past max_ctx
    no(kv.append, t, t, [(0, -1, 1)])
    no(kv.append, t, t, [(2, 0, 1)])
    no(kv.append, t, t, [(1, 0, 60)])                   # two pages are left
    no(kv.append, None, t, [(0, 0, 1)])
    no(kv.append, t, t, [(0, 0, -1)])
    no(kv.reserve, [(0, 60, 1)])
    no(kv.read, [(0, 20, 13)], t, t)                    # past its pages
    kv.reserve([(0, 32, 28)])
    no(kv.read, [(0, 60, 1)], t, t)                     # past max_ctx, within its last page
    kv.release([0], [20])
    no(kv.read, [(1, 0, 1)], t, t)
    no(kv.read, [(0, -1, 2)], t, t)
    no(kv.read, [(0, 0, 1)], t.view(-1)[1:], t)         # not 16-byte aligned
    no(si_ctx.attention_kv4, kv, dims, t, [(0, 32, 1)], t)
    no(si_ctx.attention_kv4, kv, dims, t, [(0, -2, 1)], t)
    no(si_ctx.attention_kv4, kv, dims, t, [(5, 0, 1)], t)
    no(si_ctx.attention_kv4, kv, dims, None, [(0, 0, 1)], t)
    no(si_ctx.attention_kv4, kv, dims, t.view(-1)[1:], [(0, 0, 1)], t)
    no(si_ctx.attention_kv4, kv, dims_of(12, 4, 128), t, [(0, 0, 1)], t)
    no(si_ctx.attention_kv4, kv, dims, t, [(0, 0, 1 << 22), (0, 0, 1)], t)
    no(kv.fork, [0], [1], [33])
    no(kv.fork, [0], [0], [3])
    no(kv.assign, [1], [1], [4])
    no(kv.release, [0], [-1])
    with pytest.raises(ValueError):
        kv.append(t, t, [0, 0, 1])
    with pytest.raises(ValueError):
        kv.fork([0], [1, 1], [3])
    other = sib200.Context(0, max_positions=64, head_dim=128)
    no(other.attention_kv4, kv, dims, t, [(0, 0, 1)], t)
    layer = other.layer_synth(dict(dims, hidden=1536), 1)
    okv = other.kv4(dims, 2, 128, 16, 16)
    x = torch.zeros(80, 1536, device="cuda")
    no(layer.step_dev, okv, x, [(0, 0, 65)], x)          # past the context's positions
    no(layer.step_dev, okv, x, [(0, 3, 0)], x)
    no(layer.step_dev, okv, x, [(0, 3, 1), (0, 3, 1)], x)
    no(layer.step_dev, kv, x, [(0, 3, 1)], x)
    okv.free()
    layer.free()
    other.close()
    assert kv.free_pages() == free and kv.pages(1) == []
    # nothing to do is not an error
    kv.append(t, t, [])
    kv.read([(0, 0, 0)], t, t)
    si_ctx.attention_kv4(kv, dims, t, [], t)
    si_ctx.status()
    kv.free()
