"""Rows of attention whose results are not finite, or very small in f32, which a form of their own computes again, where the keys
are shared out over workgroups and on 8-bit rows, through the C ABI against 64-bit references. Tolerances count
roundings (token_refs.py, decoder_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests.decoder_refs import held_rows, held_tolerance, split_tolerance, values_of
from tests.test_gpu_tokens import check, tensor
from tests.token_refs import attend, rounded, slot_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


@pytest.fixture(scope="module")
def stream(dev):
    return nn.Stream(dev)


def say(msg):
    print(f"[case] {msg}", flush=True)


def small(tol, keys):
    """A tolerance of results near the end of fp32's range: half its smallest step for each product and addition in the place of
    the bounds' own constant."""
    return tol - 1e-37 + 2 * keys * 2.0 ** -150


def check_odd(got, want, tol, what):
    """Finite results within tol, the others the same NaN or infinity."""
    ok = np.isfinite(want)
    np.testing.assert_array_equal(got[~ok], want[~ok], err_msg=what)
    check(got[ok], want[ok], tol[ok], what)


def all_seen(q, k, v, H, KV, scale):
    """attend() where every query sees every key, all at once, whatever the keys and values hold."""
    T, hd = q.shape[0], q.shape[1] // H
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, spread, size = (np.zeros(q.shape) for _ in range(3))
    with np.errstate(invalid="ignore"):
        for h in range(H):
            c, g = slice(h * hd, (h + 1) * hd), h * KV // H
            kc = slice(g * hd, (g + 1) * hd)
            s = q[:, c] @ k[:, kc].T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[:, c], size[:, c] = p @ v[:, kc], p @ np.abs(v[:, kc])
            spread[:, c] = (np.abs(q[:, c]) @ np.abs(k[:, kc]).T).max(-1, keepdims=True) * abs(scale)
    return out, spread, size


# ------------------------------------------------------------------ attention to an encoder's states
class States:
    """Queries and states of two sequences, kept as they come or in 8 bits."""

    def __init__(self, dev, stream, B, T, S, H, KV, hd, dtype, held, seed=0):
        rng = np.random.default_rng(seed + T)
        self.dev, self.stream, self.H, self.KV, self.hd, self.dtype, self.held = dev, stream, H, KV, hd, dtype, held
        self.q = rounded(rng.standard_normal((B, T, H * hd)), dtype)
        self.kv = [rounded(rng.standard_normal((B, S, KV * hd)), dtype) for _ in "kv"]
        self.scales = [None, None]
        if held:
            self.kv, self.scales = (list(x) for x in zip(*(held_rows(x, KV) for x in self.kv)))
        self.layer = nn.MemoryAttention(dev, H, hd, KV)
        self.clean = self.run()

    def run(self, q=None, k=None, v=None, ks=None, vs=None):
        q = self.q if q is None else q
        kv = [o if x is None else x for x, o in zip((k, v), self.kv)]
        sc = [o if x is None else x for x, o in zip((ks, vs), self.scales)]
        out = nn.Tensor(self.dev, q.shape, dtype=self.dtype)
        self.layer.forward(tensor(self.dev, q, self.dtype), *(tensor(self.dev, x, "e4m3" if self.held else self.dtype) for x in kv),
                           out, None, None, *(None if s is None else tensor(self.dev, s, "f32") for s in sc),
                           stream=self.stream)
        self.stream.sync(60000)
        return out.to_numpy()

    def check(self, got, b, keep=None, q=None, k=None, v=None, ks=None, vs=None, heads=None, tiny=False):
        """Sequence b against the formula (keep: the states that count; tiny: results are)."""
        kv = [o if x is None else x for x, o in zip((k, v), self.kv)]
        sc = [o if x is None else x for x, o in zip((ks, vs), self.scales)]
        q = (self.q if q is None else q)[b]
        with np.errstate(invalid="ignore"):
            kk, vv = ((values_of(x[b], s[b]) if self.held else x[b]) for x, s in zip(kv, sc))
        keep = slice(None) if keep is None else keep
        want, spread, size = all_seen(q, kk[keep], vv[keep], self.H, self.KV, self.hd ** -0.5)
        tol = (held_tolerance if self.held else split_tolerance)(spread, size, self.hd, len(kk), self.dtype)
        tol = small(tol, len(kk)) if tiny else tol
        cols = slice(None) if heads is None else heads
        check_odd(got[b][:, cols], want[:, cols], tol[:, cols], f"sequence {b}")

    def group(self, g):
        """The columns of the queries' heads that read head g."""
        n = self.H // self.KV * self.hd
        return slice(g * n, (g + 1) * n)


# one token and a few (k_rows.hip), many (k_memory.hip: four waves, eight waves), each with several ranges of keys
MEMORY = [(2, 1, 1600, 4, 2, 48), (2, 16, 1600, 4, 2, 64), (2, 300, 1600, 4, 2, 48), (1, 8192, 600, 8, 8, 16)]


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,S,H,KV,hd", MEMORY)
def test_memory_one_range_is_not_finite(dev, stream, B, T, S, H, KV, hd, dtype, held):
    """A value or a key of one range of many that is no number reaches all rows of its head, and nothing else."""
    say(f"memory one range {B}x{T} on {S} {dtype} held {held}")
    m = States(dev, stream, B, T, S, H, KV, hd, dtype, held)
    b, g = B - 1, KV - 1
    mine, row = m.group(g), slice(g * hd, (g + 1) * hd)
    others = [c for c in range(H * hd) if not mine.start <= c < mine.stop]

    def rest_is_clean(got):
        np.testing.assert_array_equal(got[:b], m.clean[:b])
        np.testing.assert_array_equal(got[b][:, others], m.clean[b][:, others])

    for at in (3, S // 2, S - 1):
        for bad in (np.nan, np.inf, -np.inf):
            if held:
                vs = m.scales[1].copy()
                vs[b, at, g] = bad  # e4m3 zeros times an infinite scale are NaN, the other values infinite
                change = {"vs": vs}
            else:
                v = m.kv[1].copy()
                v[b, at, g * hd + 5] = bad
                change = {"v": v}
            got = m.run(**change)
            rest_is_clean(got)
            m.check(got, b, **change)
        if held:
            k, ks = m.kv[0].copy(), m.scales[0].copy()
            x = np.ones((1, hd), np.float32)
            x[0, 2] = np.inf  # as a cache holds such a row
            with np.errstate(invalid="ignore"):
                k[b, at:at + 1, row], ks[b, at:at + 1, g:g + 1] = held_rows(x, 1)
            change = {"k": k, "ks": ks}
        else:
            k = m.kv[0].copy()
            k[b, at, g * hd + 2] = np.nan
            change = {"k": k}
        got = m.run(**change)
        rest_is_clean(got)
        assert np.isnan(got[b][:, mine]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,S,H,KV,hd", MEMORY)
def test_memory_ranges_whose_scores_are_all_minus_infinity(dev, stream, B, T, S, H, KV, hd, dtype):
    """Such a range counts for nothing beside the others, wherever it stands; where all are such, 0 / 0."""
    say(f"memory -inf ranges {B}x{T} on {S} {dtype}")
    m = States(dev, stream, B, T, S, H, KV, hd, dtype, False)
    b, q = B - 1, m.q.copy()
    q[b, :, 3::hd] = -1
    i = np.arange(S)
    for out in (i < 3 * S // 8, i >= 5 * S // 8, (i >= S // 4) & (i < 3 * S // 4), (i % 100) != 7, i >= 0):
        k = m.kv[0].copy()
        k[b, out, :hd] = np.where(np.arange(hd) == 3, np.inf, 0)
        got = m.run(q=q, k=k)
        np.testing.assert_array_equal(got[:b], m.clean[:b])
        if out.all():
            assert np.isnan(got[b][:, m.group(0)]).all()
        else:
            m.check(got, b, keep=~out, q=q, k=k, heads=m.group(0))


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("B,T,S,H,KV,hd", MEMORY)
def test_memory_very_small_results(dev, stream, B, T, S, H, KV, hd, held):
    """f32 results below 2^-109 (2^-96 on 8-bit values) keep fp32's bits, in one head beside ordinary ones."""
    say(f"memory small results {B}x{T} on {S} held {held}")
    m = States(dev, stream, B, T, S, H, KV, hd, "f32", held)
    b = B - 1
    if held:
        vs = m.scales[1].copy()
        vs[b, :, 0] *= np.float32(1e-30)
        change = {"vs": vs}
    else:
        v = m.kv[1].copy()
        v[b, :, :hd] *= np.float32(1e-34)
        change = {"v": v}
    got = m.run(**change)
    m.check(got, b, tiny=True, **change)
    np.testing.assert_array_equal(got[:b], m.clean[:b])


# ---------------------------------------------------------------------- steps on 8-bit caches
class Steps:
    """Three streams' caches, wrapped several times, and their next T tokens."""

    def __init__(self, dev, stream, T, H, KV, hd, left, sinks, dtype, seed=0):
        rng = np.random.default_rng(seed + T)
        self.dev, self.stream, self.T, self.H, self.KV, self.hd = dev, stream, T, H, KV, hd
        self.left, self.sinks, self.dtype, self.slots = left, sinks, dtype, sinks + left + T + 2
        self.pos = [5 * self.slots + 11, left // 3, 2 * self.slots]
        B, w = len(self.pos), KV * hd
        self.q = rounded(rng.standard_normal((B, T, H * hd)), dtype)
        self.new = [rounded(rng.standard_normal((B, T, w)), dtype) for _ in "kv"]
        self.old = [held_rows(rng.standard_normal((B, self.slots, w)), KV) for _ in "kv"]
        self.layer = nn.WindowAttention(dev, H, hd, KV, left, 0, sinks)

    def run(self, new, old):
        out = nn.Tensor(self.dev, self.q.shape, dtype=self.dtype)
        c, s = [tensor(self.dev, x, "e4m3") for x, _ in old], [tensor(self.dev, x, "f32") for _, x in old]
        self.layer.step(tensor(self.dev, self.q, self.dtype), *(tensor(self.dev, x, self.dtype) for x in new),
                        tensor(self.dev, np.array(self.pos), "i32"), *c, out, None, self.stream, *s)
        self.stream.sync(60000)
        return out.to_numpy(), [x.to_numpy() for x in (*c, *s)]

    def slot(self, p):
        return slot_of(p, self.sinks, self.slots)

    def want(self, b, new, old):
        """(result, tolerance) of stream b."""
        p = self.pos[b]
        first = max(0, p - self.left)
        told = list(range(min(self.sinks, first))) + list(range(first, p + self.T))
        at = [self.slot(i) for i in told[:len(told) - self.T]]
        with np.errstate(invalid="ignore"):
            k, v = (np.concatenate([values_of(x[b, at], s[b, at]), values_of(*held_rows(n[b], self.KV))])
                    for (x, s), n in zip(old, new))
            mine, key = np.arange(p, p + self.T)[:, None], np.array(told)[None]
            seen = (key <= mine) & ((key >= mine - self.left) | (key < self.sinks))
            want, spread, size = attend(self.q[b], k, v, seen, self.H, self.KV, self.hd ** -0.5)
        return want, held_tolerance(spread, size, self.hd, len(told), self.dtype)

    def check(self, new, old, clean, odd, tiny=False):
        """The streams of `odd` against the formula, the others bit for bit; the new rows in their slots."""
        got, cache = self.run(new, old)
        for b in range(len(self.pos)):
            if b in odd:
                want, tol = self.want(b, new, old)
                check_odd(got[b], want, small(tol, self.slots) if tiny else tol, f"stream {b}")
            else:
                np.testing.assert_array_equal(got[b], clean[b])
            at = [self.slot(self.pos[b] + i) for i in range(self.T)]
            for c in (0, 1):
                with np.errstate(invalid="ignore"):
                    x, s = held_rows(new[c][b], self.KV)
                np.testing.assert_array_equal(cache[c][b, at], x)
                np.testing.assert_array_equal(cache[2 + c][b, at], s)
        return got


STEPS = [(1, 4, 2, 48, 700, 3), (16, 4, 2, 64, 700, 3), (3, 8, 8, 128, 300, 0), (40, 4, 1, 32, 90, 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,H,KV,hd,left,sinks", STEPS)
def test_window_step_held_rows_that_are_not_finite(dev, stream, T, H, KV, hd, left, sinks, dtype):
    """A NaN or an infinity in a row of the cache or among the call's own rows, a key's or a value's, reaches the tokens that see
    it, in its head: the other heads and streams keep their bits, earlier tokens of the call their results."""
    say(f"8-bit step not finite T {T} heads {H}/{KV} hd {hd} left {left} sinks {sinks} {dtype}")
    m = Steps(dev, stream, T, H, KV, hd, left, sinks, dtype)
    clean, _ = m.run(m.new, m.old)
    for b in range(len(m.pos)):
        check_odd(clean[b], *m.want(b, m.new, m.old), f"clean stream {b}")
    g, n = KV - 1, H // KV * hd
    others = [c for c in range(H * hd) if not g * n <= c < (g + 1) * n]
    for b in (0, 1):
        p = m.pos[b]
        tokens = [p - 1, max(0, p - left) + T // 2, p + T // 2, p + T - 1] + ([1] if sinks else [])
        for at in tokens:
            for c in (0, 1):
                for bad in (np.nan, np.inf):
                    new, old = [x.copy() for x in m.new], [(x.copy(), s.copy()) for x, s in m.old]
                    if at >= p:
                        new[c][b, at - p, g * hd + 1] = bad
                    else:
                        row = values_of(old[c][0][b, m.slot(at)][None], old[c][1][b, m.slot(at)][None])
                        row[0, g * hd + 1] = bad
                        with np.errstate(invalid="ignore"):
                            x, s = held_rows(row[:, g * hd:(g + 1) * hd], 1)
                        old[c][0][b, m.slot(at), g * hd:(g + 1) * hd], old[c][1][b, m.slot(at), g] = x[0], s[0, 0]
                    got = m.check(new, old, clean, (b,))
                    np.testing.assert_array_equal(got[b][:, others], clean[b][:, others])


@pytest.mark.parametrize("T,H,KV,hd,left,sinks", STEPS)
def test_window_step_held_very_small_results(dev, stream, T, H, KV, hd, left, sinks):
    """f32 values of about 1e-30, kept and new: results below 2^-96 keep fp32's bits."""
    say(f"8-bit step small results T {T} heads {H}/{KV} hd {hd} left {left} sinks {sinks}")
    m = Steps(dev, stream, T, H, KV, hd, left, sinks, "f32")
    clean, _ = m.run(m.new, m.old)
    new, old = [m.new[0], m.new[1].copy()], [m.old[0], (m.old[1][0], m.old[1][1].copy())]
    new[1][:2] *= np.float32(1e-30)
    old[1][1][:2] *= np.float32(1e-30)
    m.check(new, old, clean, (0, 1), tiny=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cache_rows_near_the_largest(dev, stream, dtype):
    """Rows whose largest value's reciprocal is no normal number, and steps that see them."""
    say(f"8-bit rows near the largest {dtype}")
    m = Steps(dev, stream, 2, 4, 2, 48, 60, 1, dtype)
    for size in (9e37, 3.3e38):
        x = rounded(np.sign(m.new[1]) * np.minimum(np.abs(m.new[1]), 1) * size, dtype)
        want, ws = held_rows(x, 2)
        _, cache = m.run([m.new[0], x], m.old)
        for b in range(3):
            at = [m.slot(m.pos[b] + i) for i in range(2)]
            np.testing.assert_array_equal(cache[1][b, at], want[b])
            np.testing.assert_array_equal(cache[3][b, at], ws[b])
