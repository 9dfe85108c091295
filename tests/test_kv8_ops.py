"""The attention over caches of 8 bits (include/bitnet_hip.h section 5: kv8_rows, kv8_read, kv8_step, kv8_prefill), one operator at a time through the C ABI and then together, against f64
numpy (tests/kv8_util.py).

Tolerances.  A number of the cache is off by half a step of its scale at most, and by what 32 bits lose ahead of it (1e-5 of the largest).  STEP: a step's chain is 32 bits wide (norm, factor
and scale: four roundings of 2^-24 on a score, of magnitude up to ten here: 2.4e-6), queries have 23 bits of their largest element and weights 22: together under 5e-6 of a weight, errors of
different weights independent; twice that is allowed.  PROMPT: a weight is an f16 (2^-12), a query 15 bits of its largest element (a few 2^-16 of a score of up to ten: 5e-4): 2^-10; and the
output a bf16 (2^-9 at most).  Two maps: what their difference makes of either's error (kv8_util.Attention.want)."""
import numpy as np
import pytest

from tests import kv8_util as kv
from tests import stack_util as u

pytestmark = pytest.mark.gpu
STEP, PROMPT = 1e-5, (2.0 ** -10, 2.0 ** -9)
f64 = np.float64


def as_bf16(t):
    import torch

    return t.bfloat16().view(torch.int16)


# heads, kv heads, dim, vdim, maps
SHAPES = [(4, 2, 24, 40, 2), (6, 6, 128, 128, 2), (20, 1, 64, 100, 2), (8, 2, 96, 64, 1), (2, 1, 200, 256, 2), (5, 1, 40, 16, 1), (34, 2, 16, 24, 2), (8, 2, 128, 128, 1), (3, 3, 64, 64, 1),
          (16, 2, 256, 160, 1)]
# what else an attention can have, on heads that take it
OPTIONS = [dict(rot=16), dict(rot=24, window=37), dict(chunk=50, sink=True, gate="heads", rot=8), dict(far=True, gate="columns", window=100), dict(keys_as_values=True, normed=False, sink=True),
           dict(normed=False, far=True), dict(gate="columns")]


# ---- writing ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("n0,n", [(0, 1), (31, 1), (5, 2), (31, 2), (0, 32), (7, 33), (17, 130), (64, 64), (3, 300)])
@pytest.mark.parametrize("shape", SHAPES)
def test_written_bit_by_bit(hip, pkg, shape, n0, n, f32):
    """keys and values without anything ahead of them: numbers and scales as the rule gives them, everything else as it was"""
    t = kv.Attention(pkg, n0 + n, *shape, normed=False, f32=f32, fill=77, scale=5.0)
    _, q = t.fill(hip, n0, n0 + n)
    k, v, ks, vs = t.cache.host()
    for got, scales, x in ((k, ks, t.k), (v, vs, t.v)):
        numbers, scale = kv.numbers_of(x)
        assert np.array_equal(got[..., n0:n0 + n, :], numbers[..., n0:n0 + n, :]) and np.array_equal(scales[..., n0:n0 + n], scale[..., n0:n0 + n])
        assert (got[..., :n0, :] == 77).all() and (got[..., n0 + n:, :] == 77).all() and (scales[..., :n0] == 5).all() and (scales[..., n0 + n:] == 5).all()
    got = u.host(q).reshape(n, -1, t.dimp)
    assert u.rms_error(got[..., :t.dim], t.q[n0:]) < (1e-6 if f32 else 2.0 ** -8) and not got[..., t.dim:].any()


@pytest.mark.parametrize("shape,n0,n", [((64, 64, 32, 32, 1), 5, 1100), ((30, 30, 24, 40, 2), 32, 2300), ((40, 40, 200, 200, 1), 19, 1700)])
def test_many_tokens_of_many_heads(hip, pkg, shape, n0, n):
    """values by pieces of 32 positions"""
    test_written_bit_by_bit(hip, pkg, shape, n0, n, False)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("options", [dict(), dict(rot=16), dict(taps=3), dict(taps=5, rot=24), dict(taps=1, keys_as_values=True), dict(keys_as_values=True, rot=4)])
@pytest.mark.parametrize("shape", [(6, 2, 24, 24, 1), (4, 2, 128, 128, 1), (2, 1, 200, 200, 1), (4, 2, 64, 100, 2)])
def test_written_behind_norms_and_convolutions(hip, pkg, shape, options, f32):
    if shape[4] == 2 and options.get("keys_as_values"):
        pytest.skip("two maps have values of their own")
    t = kv.Attention(pkg, 210, *shape, f32=f32, **options)
    for n0, n1 in ((0, 3), (3, 4), (4, 130), (130, 210)):
        rows, q = t.fill(hip, n0, n1)
        got = u.host(q).reshape(n1 - n0, -1, t.dimp)
        assert u.rms_error(got[..., :t.dim], t.q[n0:n1]) < (3e-6 if f32 else 2.0 ** -8)
        assert np.array_equal(u.host(rows), t.rows[n0:n1])
    k, v, ks, vs = t.cache.host()
    for got, scales, x in ((k, ks, t.k), (v, vs, t.v)):
        got, scales = got[..., :210, :].astype(f64), scales[..., :210].astype(f64)
        largest = np.abs(x).max(-1)
        assert np.abs(scales * 127 / largest - 1).max() < 1e-5
        assert (np.abs(got * scales[..., None] - x) <= scales[..., None] * 0.5 + 1e-5 * largest[..., None]).all()


def test_queries_in_place_and_rows_further_apart(hip, pkg):
    t = kv.Attention(pkg, 40, 5, 1, 40, 16)
    rows = np.full((40, t.ld + 8), 7, np.float32)
    rows[:, :t.ld] = t.rows
    d = u.dev_bf16(rows)
    pos = u.dev(np.array([0], np.int32))
    hip.kv8_rows_dev(t.attn, t.cache.ks, t.cache.vs, d, t.ld + 8, False, pos, 40)
    got, nq = u.host(d), t.heads * t.dimp
    assert np.array_equal(got[:, nq:], rows[:, nq:]) and u.rms_error(got[:, :nq].reshape(40, 5, -1)[..., :40], t.q) < 2.0 ** -8
    before = t.cache.host()
    t.fill(hip, 0, 40)
    assert all(np.array_equal(a, b) for a, b in zip(before, t.cache.host()))


def test_values_that_no_scale_fits(hip, pkg):
    """zeros, tiny and huge numbers, infinities and NaN: zeros, numbers or no numbers, each position by itself"""
    t = kv.Attention(pkg, 40, 2, 1, 64, 64, normed=False, f32=True, seed=3)
    nq, nk = 2 * 64, 64
    for i, x in enumerate((0.0, 1e-37, 1e-45, 1.4e-36, 1.6e-36, 1e30, 3e38, np.inf, -np.inf, np.nan)):
        t.rows[i, nq:nq + 2 * nk] *= 0
        t.rows[i, nq + 5] = t.rows[i, nq + nk + 60] = x
        t.rows[i, nq + 6] = t.rows[i, nq + nk + 3] = 0 if not np.isfinite(x) else -x / 3
    t.fill(hip, 0, 40)
    k, v, ks, vs = t.cache.host()
    for got, scales, first in ((k[0, 0], ks[0, 0], nq), (v[0], vs[0], nq + nk)):
        numbers, scale = kv.numbers_of(t.rows[:, first:first + nk])
        assert np.array_equal(got[:40], numbers) and np.array_equal(scales[:40], scale, equal_nan=True)
        assert np.isnan(scales[7:10]).all() and (scales[:4] == 0).all() and (scales[4:7] > 0).all()


@pytest.mark.parametrize("shape", SHAPES[:6])
def test_portions_and_steps_write_the_same(hip, pkg, shape):
    """the cache is a function of the tokens: at once, in portions, and one by one"""
    n = 70
    whole, cut, steps = (kv.Attention(pkg, n, *shape, f32=True, rot=8) for _ in range(3))
    whole.fill(hip, 0, n)
    for n0, n1 in ((0, 1), (1, 30), (30, 33), (33, 70)):
        cut.fill(hip, n0, n1)
    for i in range(n):
        steps.step(hip, i)
    a = whole.cache.host()
    assert all(np.array_equal(x, y) for x, y in zip(a, cut.cache.host()))
    for x, y, held in zip(a[2:], steps.cache.host()[2:], (whole.k, whole.v)):  # (a step sums a norm in another order)
        assert np.allclose(x, y, rtol=1e-6, atol=0)
    for x, y in zip(a[:2], steps.cache.host()[:2]):
        assert np.abs(x.astype(int) - y).max() <= 1 and (x != y).mean() < 1e-3


def test_a_position_written_again(hip, pkg):
    t, other = (kv.Attention(pkg, 50, 4, 2, 24, 40, 2, seed=s) for s in (0, 1))
    other.fill(hip, 0, 50)
    t.attn.kcache, t.attn.vcache, cache, t.cache = other.cache.k.data_ptr(), other.cache.v.data_ptr(), t.cache, other.cache
    t.fill(hip, 10, 37)
    k, v, ks, vs = t.cache.host()
    t.attn.kcache, t.attn.vcache, t.cache = cache.k.data_ptr(), cache.v.data_ptr(), cache
    t.fill(hip, 10, 37)
    assert all(np.array_equal(a[..., 10:37, :], b[..., 10:37, :]) for a, b in zip((k, v), t.cache.host()))
    other.fill(hip, 10, 37)
    again = other.cache.host()
    fresh = kv.Attention(pkg, 50, 4, 2, 24, 40, 2, seed=1)
    fresh.fill(hip, 0, 50)
    assert all(np.array_equal(a, b) for a, b in zip(again, fresh.cache.host()))


# ---- reading back -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("first,n", [(0, 1), (31, 1), (31, 2), (0, 384), (5, 300), (96, 33), (383, 1)])
@pytest.mark.parametrize("shape", SHAPES)
def test_read_back(hip, pkg, shape, first, n, f32):
    import torch

    heads, g, dim, vdim, maps = shape
    t = kv.Attention(pkg, 384, heads, g, dim, vdim, maps)
    gen = torch.Generator(device="cuda").manual_seed(n)
    c = t.cache
    for x in (c.k, c.v):
        x.copy_(torch.randint(-127, 128, x.shape, generator=gen, device="cuda", dtype=torch.int8))
    for x in (c.ks, c.vs):
        x.copy_(torch.rand(x.shape, generator=gen, device="cuda"))
    new = torch.float32 if f32 else torch.bfloat16
    keys, values = torch.full((g, maps, n, t.dimp), 3, dtype=new, device="cuda"), torch.full((g, n, t.vdimp), 3, dtype=new, device="cuda")
    hip.kv8_read_dev(t.attn, c.ks, c.vs, first, n, keys, values, f32)
    k, v, ks, vs = c.host()
    for got, numbers, scale in ((keys, k, ks), (values, v, vs)):
        want = numbers[..., first:first + n, :].astype(np.float32) * scale[..., first:first + n, None]
        assert np.array_equal(got.float().cpu().numpy(), want if f32 else u.rounded(want))
    for which in (0, 1):
        a, b = torch.zeros_like(keys), torch.zeros_like(values)
        hip.kv8_read_dev(t.attn, c.ks, c.vs, first, n, None if which else a, b if which else None, f32)
        assert bool((a == (0 * keys if which else keys)).all()) and bool((b == (values if which else 0 * values)).all())


# ---- steps --------------------------------------------------------------------------------------------------------------
def stepped(hip, t, i):
    if i:
        t.fill(hip, 0, i)
    before = [a.copy() for a in t.cache.host()]
    out = t.step(hip, i)
    t.check(out, t.want(t.q[i:i + 1], i), STEP)
    for a, b in zip(before, t.cache.host()):  # nothing but the position
        axis = b.ndim - 2 if a.dtype == np.int8 else b.ndim - 1
        assert np.delete(a, i, axis).tobytes() == np.delete(b, i, axis).tobytes()  # (some are no numbers)
    numbers, scale = kv.numbers_of(t.k[..., i, :])
    assert np.allclose(t.cache.host()[2][..., i], scale, rtol=1e-5) and np.abs(t.cache.host()[0][..., i, :].astype(int) - numbers).max() <= 1
    if t.maps == 2:  # (keys of another layer: one map)
        return
    kept = t.cache.host()
    t.check(t.step(hip, i, queries_only=True), t.want(t.q[i:i + 1], i), STEP)
    assert all(a.tobytes() == b.tobytes() for a, b in zip(kept, t.cache.host()))


@pytest.mark.parametrize("n", [1, 2, 32, 33, 64, 65, 127, 128, 129, 257, 700])
@pytest.mark.parametrize("shape", SHAPES)
def test_step(hip, pkg, shape, n):
    """garbage behind the positions written, scales that are no numbers among it"""
    stepped(hip, kv.Attention(pkg, n, *shape, fill=-128, scale=np.nan), n - 1)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("n", [1, 33, 100, 129, 300])
@pytest.mark.parametrize("shape", [(6, 2, 24, 24), (4, 4, 128, 128), (20, 1, 96, 96), (2, 1, 200, 200)])
def test_step_with_everything_else(hip, pkg, shape, n, options):
    stepped(hip, kv.Attention(pkg, n, *shape, fill=99, scale=np.inf, **options), n - 1)


@pytest.mark.parametrize("n,window", [(17000, 0), (40000, 0), (40000, 700), (16513, 16384)])
def test_step_behind_many_keys(hip, pkg, n, window):
    """records of several tiles; sharp scores"""
    t = kv.Attention(pkg, n, 3, 1, 64, 64, window=window, sharp=3.0)
    t.fill(hip, 0, n - 1)
    t.check(t.step(hip, n - 1), t.want(t.q[n - 1:], n - 1), STEP * 3)


@pytest.mark.parametrize("shape,n", [((20, 20, 32, 32, 1), 8000), ((10, 5, 64, 64, 1), 16200), ((3, 3, 200, 200, 1), 12800), ((12, 12, 32, 64, 2), 5700), ((40, 40, 64, 64, 1), 13 * 128 + 1)])
def test_step_of_more_records_than_the_chip_holds_at_once(hip, pkg, shape, n):
    """neighbouring records become one; what lay in their places is gone"""
    t = kv.Attention(pkg, n, *shape)
    t.fill(hip, 0, n - 1)
    scratch = u.zeros_f32(hip.gqa_scratch_bytes(t.heads, t.maps, t.vdimp, 1) // 4)
    scratch.fill_(np.nan)
    t.check(t.step(hip, n - 1, scratch=scratch), t.want(t.q[n - 1:], n - 1), STEP * 3)


@pytest.mark.parametrize("spread", [1e-30, 1e-3, 1e3, 1e30])
def test_values_of_very_different_size(hip, pkg, spread):
    """scales grow and shrink by the token: what is large decides, whatever came ahead of it"""
    for n in (40, 300):
        t = kv.Attention(pkg, n, 4, 2, 64, 64, normed=False, f32=True)
        at = 4 * t.dimp + 2 * t.dimp
        t.rows[::7, at:at + 2 * t.vdimp] *= np.float32(spread)
        t.convolved = t.rows[:, :t.channels].astype(f64)
        t.fill(hip, 0, n - 1)
        t.check(t.step(hip, n - 1), t.want(t.q[n - 1:], n - 1), STEP)
        _, q = t.fill(hip, 0, n)
        qb = as_bf16(q)
        t.check(t.prompt(hip, qb, 0, n), t.want(u.host(qb).reshape(n, -1, t.dimp)[..., :t.dim], 0), *PROMPT)


@pytest.mark.parametrize("up", [90, -90])
def test_queries_and_keys_of_opposite_size(hip, pkg, up):
    """powers of two that take each other away: the same scores"""
    n = 200
    t = kv.Attention(pkg, n, 4, 2, 64, 64, normed=False, f32=True)
    heads = 4 * t.dimp
    t.rows[:, :heads] *= np.float32(2.0 ** up)
    t.rows[:, heads:heads + 2 * t.dimp] *= np.float32(2.0 ** -up)
    t.convolved = t.rows[:, :t.channels].astype(f64)
    t.q *= 2.0 ** up
    t.fill(hip, 0, n - 1)
    t.check(t.step(hip, n - 1), t.want(t.q[n - 1:], n - 1), STEP)
    _, q = t.fill(hip, 0, n)
    qb = as_bf16(q)
    t.check(t.prompt(hip, qb, 0, n), t.want(u.host(qb).reshape(n, -1, t.dimp)[..., :t.dim], 0), *PROMPT)


# ---- prompts ------------------------------------------------------------------------------------------------------------
def prompted(hip, t, n0, n):
    if n0:
        t.fill(hip, 0, n0)
    _, q = t.fill(hip, n0, n)
    want = t.want(u.host(q).reshape(n - n0, -1, t.dimp)[..., :t.dim], n0)
    outs = [t.prompt(hip, q, n0, n, split) for split in (True, False)]
    for out in outs:
        t.check(out, want, *PROMPT)


@pytest.mark.parametrize("n,nq", [(1, 1), (2, 2), (63, 63), (65, 65), (128, 128), (129, 2), (200, 200), (333, 70), (600, 5)])
@pytest.mark.parametrize("shape", SHAPES)
def test_prompt(hip, pkg, shape, n, nq):
    prompted(hip, kv.Attention(pkg, n, *shape, fill=-128, scale=np.nan), n - nq, n)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("n,nq", [(1, 1), (130, 130), (333, 40)])
@pytest.mark.parametrize("shape", [(6, 2, 24, 24), (4, 4, 128, 128), (20, 1, 96, 96), (2, 1, 200, 200)])
def test_prompt_with_everything_else(hip, pkg, shape, n, nq, options):
    prompted(hip, kv.Attention(pkg, n, *shape, fill=99, scale=np.inf, **options), n - nq, n)


@pytest.mark.parametrize("shape", [(8, 2, 128, 128, 1), (4, 1, 64, 128, 2), (9, 3, 64, 64, 1), (2, 1, 256, 256, 1)])
@pytest.mark.parametrize("n,nq", [(1100, 1100), (2500, 40), (2500, 130)])
def test_long_prompts(hip, pkg, shape, n, nq):
    """one group and two, stretches and whole walks; a sample of the queries by definition"""
    t = kv.Attention(pkg, n, *shape, rot=16, sharp=2.0)
    if n > nq:
        t.fill(hip, 0, n - nq)
    _, q = t.fill(hip, n - nq, n)
    some = np.unique(np.linspace(0, nq - 1, 23).astype(int))
    held, qh = t.cache.held(), u.host(q).reshape(nq, -1, t.dimp)[..., :t.dim]
    want = np.concatenate([t.want(qh[i:i + 1], n - nq + i, held) for i in some])
    for split in (True, False):
        t.check(u.dev_f32(u.host(t.prompt(hip, q, n - nq, n, split))[some]), want, *PROMPT)


# ---- what must not spread -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("what", ["key", "value"])
def test_a_token_without_numbers_reaches_who_sees_it(hip, pkg, what):
    """a NaN in one token's key or value: earlier queries and those whose window has passed keep their outputs, the others have none"""
    n, bad, window = 200, 70, 60
    t = kv.Attention(pkg, n, 4, 2, 64, 64, window=window, f32=True)
    clean = kv.Attention(pkg, n, 4, 2, 64, 64, window=window, f32=True)
    at = 4 * t.dimp + (0 if what == "key" else 2 * t.dimp)
    for a in (t, clean):  # (not the largest of its tile: what the others' weights are brought to stays the same)
        a.rows[bad, 6 * t.dimp:8 * t.dimp] *= 0.01
        a.convolved[bad, 6 * t.dimp:8 * t.dimp] *= 0.01
    t.rows[bad, at + 3] = t.convolved[bad, at + 3] = np.nan  # (the first kv head's: heads 0 and 1)
    outs = []
    for a in (t, clean):
        _, q = a.fill(hip, 0, n)
        outs.append(u.host(a.prompt(hip, as_bf16(q), 0, n)).reshape(n, 4, 64))
    sees = np.arange(n)
    sees = (sees >= bad) & (sees < bad + window)
    assert np.isnan(outs[0][sees][:, :2]).all()
    assert np.array_equal(outs[0][~sees], outs[1][~sees]) and np.array_equal(outs[0][:, 2:], outs[1][:, 2:])
    for i in (bad - 1, bad, bad + window - 1, bad + window, n - 1):
        got, want = (u.host(a.step(hip, i)).reshape(4, 64) for a in (t, clean))
        assert np.isnan(got[:2]).all() if sees[i] else np.array_equal(got, want)
        assert np.array_equal(got[2:], want[2:])


def test_queries_without_numbers(hip, pkg):
    """a query that is not finite has no output, one of zeros weighs all keys alike, and no other query notices"""
    n = 150
    t = kv.Attention(pkg, n, 4, 2, 64, 64, normed=False, f32=True)
    _, q = t.fill(hip, 0, n)
    q[20, 64:128] = float("inf")
    q[40, 3] = float("nan")
    q[60] = 0
    q = as_bf16(q)
    got = u.host(t.prompt(hip, q, 0, n)).reshape(n, 4, 64)
    assert np.isnan(got[20, 1]).all() and np.isnan(got[40, 0]).all()
    got[20, 1] = got[40, 0] = 0
    qh = u.host(q).reshape(n, 4, 64)
    qh[20, 1] = qh[40, 0] = 0
    want = t.want(qh, 0)
    want[20, 1] = want[40, 0] = 0
    t.check(u.dev_f32(got), want, *PROMPT)
    mean = t.cache.held()[1][0, :61].mean(0)
    assert u.rms_error(got[60, 0], mean) < sum(PROMPT)


@pytest.mark.parametrize("sink", [-60.0, 12.0, 20.0, 60.0])
def test_sinks_far_from_every_score(hip, pkg, sink):
    """one far above leaves small outputs, to as many bits as others"""
    n = 300
    t = kv.Attention(pkg, n, 6, 2, 64, 64, sink=True)
    t.sink[:] = sink + np.arange(6)
    t.keep.append(u.dev_f32(t.sink))
    t.attn.sink = t.keep[-1].data_ptr()
    _, q = t.fill(hip, 0, n)
    want = t.want(u.host(q).reshape(n, -1, t.dimp)[..., :t.dim], 0)
    for split in (True, False):
        t.check(t.prompt(hip, q, 0, n, split), want, *PROMPT)
    t.check(t.step(hip, n - 1), t.want(t.q[n - 1:], n - 1), STEP)


# ---- together -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(20, 5, 128, 128, 1), (12, 3, 64, 128, 2), (6, 2, 96, 96, 1)])
def test_a_sequence_as_it_is_used(hip, pkg, shape):
    """two portions, then steps; the outputs against f64 over the cache and over keys and values that were never rounded, and the cache read back"""
    import torch

    n = 330
    t = kv.Attention(pkg, n, *shape, rot=32, f32=False)
    for n0, n1 in ((0, 130), (130, 300)):
        _, q = t.fill(hip, n0, n1)
        out = t.prompt(hip, q, n0, n1)
        t.check(out, t.want(u.host(q).reshape(n1 - n0, -1, t.dimp)[..., :t.dim], n0), *PROMPT)
    for i in range(300, n):
        out = t.step(hip, i)
        t.check(out, t.want(t.q[i:i + 1], i), STEP)
        # A number is off by a step / sqrt(12), steps being independent: a score by |q| (a key's scale) / sqrt(12), which is what a weight is off by, and a value by its scale / sqrt(12).
        # The output, a sum of values with independent errors, is off by both together, relative to the values; three times the largest of either is allowed.
        _, _, ks, vs = t.cache.host()
        off = 3 / np.sqrt(12) * (np.linalg.norm(t.q[i], axis=-1).max() * ks[..., :i + 1].max() + (vs[:, :i + 1] / np.sqrt((t.v[:, :i + 1] ** 2).mean(-1))).max())
        t.check(out, t.want(t.q[i:i + 1], i, (t.k, t.v)), off)
    keys, values = torch.zeros(shape[1], shape[4], n, t.dimp, device="cuda"), torch.zeros(shape[1], n, t.vdimp, device="cuda")
    hip.kv8_read_dev(t.attn, t.cache.ks, t.cache.vs, 0, n, keys, values, True)
    for got, x in ((keys, t.k), (values, t.v)):
        assert (np.abs(got.cpu().numpy() - x) <= np.abs(x).max(-1, keepdims=True) * (0.5 / 127 + 1e-5)).all()


def test_two_streams_and_a_graph(hip, pkg):
    """a captured step and prompt, replayed at other positions among eager work on other streams, give what eager calls give; two captures with scratch of their own do not meet"""
    import torch

    n = 260
    a, b = (kv.Attention(pkg, n, 8, 2, 128, 128, rot=64, f32=True, seed=s) for s in (0, 1))
    side = torch.cuda.Stream()
    held = []
    for t in (a, b):
        t.fill(hip, 0, n)
        held.append([x.clone() for x in (t.cache.k, t.cache.v, t.cache.ks, t.cache.vs)])
    positions = [200, 129, 64, 259, 0]
    for t in (a, b):  # (as steps leave the positions)
        for i in positions:
            t.step(hip, i)
    want = [[u.host(t.step(hip, i)).copy() for i in positions] for t in (a, b)]
    graphs = []
    for t in (a, b):
        pos, row = u.dev(np.array([0], np.int32)), u.zeros_f32(t.ld)
        scratch, out = u.zeros_f32(hip.gqa_scratch_bytes(8, 1, 128, 1) // 4), u.zeros_f32(1, 8 * 128)
        q, prompt = u.zeros_bf16(n, 8 * 128), u.zeros_bf16(n, 8 * 128)
        q.copy_(as_bf16(u.dev_f32(t.q.reshape(n, -1))))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s = torch.cuda.current_stream().cuda_stream
            hip.kv8_step_dev(t.attn, t.cache.ks, t.cache.vs, row, pos, scratch, stream=s)
            hip.gqa_merge_dev(t.attn, pos, 0, 1, scratch, out, 8 * 128, False, stream=s)
            hip.kv8_prefill_dev(t.attn, t.cache.ks, t.cache.vs, q, q.shape[1], n, n, prompt, 8 * 128, stream=s)
        graphs.append((graph, pos, row, out, q, prompt, scratch))  # (all of them live as long as the graph)
    eager = [u.host(t.prompt(hip, g[4], 0, n, split=False)).copy() for t, g in zip((a, b), graphs)]
    for k, i in enumerate(positions):
        for t, (_, pos, row, *_) in zip((a, b), graphs):
            pos.fill_(i)
            row.copy_(u.dev_f32(t.rows[i]))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for w in range(2):
            assert np.array_equal(u.host(graphs[w][3]), want[w][k]), (w, i)
            assert np.array_equal(u.host(graphs[w][5]), eager[w]), (w, i)
        t = (a, b)[k & 1]
        u.host(t.step(hip, positions[k - 1]))
    for t, before in zip((a, b), held):
        t.fill(hip, 0, n)
        assert all(bool((x == y).all()) for x, y in zip(before, (t.cache.k, t.cache.v, t.cache.ks, t.cache.vs)))


def test_caches_past_two_gigabytes(hip, pkg):
    """8 heads of 256 columns at a capacity of 1310720: offsets of the last head pass 32 bits"""
    import torch

    cap, kvh, heads = 1310720, 8, 8
    base = cap - 700
    small = kv.Attention(pkg, 640, heads, kvh, 256, 256, window=200, f32=True)
    t = kv.Attention(pkg, 640, heads, kvh, 256, 256, window=200, f32=True)
    big = kv.Cache(kvh, 1, cap, 256, 256)
    factor = torch.zeros(cap, device="cuda")
    factor[base:base + 640] = t.keep[2][:640]
    t.attn.capacity, t.attn.kcache, t.attn.vcache, t.attn.q_factor = cap, big.k.data_ptr(), big.v.data_ptr(), factor.data_ptr()
    rows, pos, q = t.put(t.rows), u.dev(np.array([base], np.int32)), u.zeros_f32(640, heads * 256)
    hip.kv8_rows_dev(t.attn, big.ks, big.vs, rows, t.ld, True, pos, 640, q, q.shape[1])
    _, qs = small.fill(hip, 0, 640)
    assert bool((q == qs).all())
    got, want = u.zeros_bf16(300, heads * 256), u.zeros_bf16(300, heads * 256)
    hip.kv8_prefill_dev(t.attn, big.ks, big.vs, as_bf16(q)[340:].contiguous(), heads * 256, base + 640, 300, got, heads * 256)
    hip.kv8_prefill_dev(small.attn, small.cache.ks, small.cache.vs, as_bf16(qs)[340:].contiguous(), heads * 256, 640, 300, want, heads * 256)
    assert u.rms_error(u.host(got), u.host(want)) < sum(PROMPT)  # (tiles of keys begin elsewhere)
    keys, values = torch.zeros(kvh, 1, 640, 256, device="cuda"), torch.zeros(kvh, 640, 256, device="cuda")
    hip.kv8_read_dev(t.attn, big.ks, big.vs, base, 640, keys, values, True)
    k, v = small.cache.held()
    assert u.rms_error(keys.cpu().numpy(), k) < 1e-7 and u.rms_error(values.cpu().numpy(), v) < 1e-7
    scratch, out = u.zeros_f32(hip.gqa_scratch_bytes(heads, 1, 256, 1) // 4), u.zeros_f32(1, heads * 256)
    at = u.dev(np.array([base + 639], np.int32))
    hip.kv8_step_dev(t.attn, big.ks, big.vs, u.dev_f32(t.rows[639]), at, scratch)
    hip.gqa_merge_dev(t.attn, at, 0, 1, scratch, out, heads * 256, False)
    assert u.rms_error(u.host(out), u.host(small.step(hip, 639))) < 2 * STEP


def test_more_than_two_to_the_31_pieces_read_back(hip, pkg):
    """a cache whose keys are more than 2^31 pieces of sixteen bytes, read in one call"""
    import torch

    n = 2 ** 27 + 72
    if torch.cuda.mem_get_info()[0] < 3.3 * 256 * n:
        pytest.skip("wants 110 GB")
    cap = u.up_to(n, 128)
    keys, scales = torch.zeros(cap, 256, dtype=torch.int8, device="cuda"), torch.zeros(cap, device="cuda")
    some = torch.tensor([0, 1, 15, 16, 17, 255, 4099, 2 ** 26 + 3, 2 ** 27 - 1, 2 ** 27, 2 ** 27 + 1, n - 17, n - 1], device="cuda")
    numbers = torch.randint(-127, 128, (len(some), 256), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda", dtype=torch.int8)
    keys[some], scales[some] = numbers, torch.arange(1, len(some) + 1, device="cuda") * 0.5
    attn = pkg.Gqa(1, 1, 1, 256, 256, 256, 256, cap, 1e-5, 0.0, 1.0, 0, 0, scales.data_ptr(), keys.data_ptr(), keys.data_ptr())
    out = torch.full((n + 1, 256), 3, dtype=torch.bfloat16, device="cuda")
    hip.kv8_read_dev(attn, scales, scales, 0, n, out, None, False)
    assert bool((out[some].float() == (numbers.float() * scales[some, None]).bfloat16().float()).all()) and bool((out[n] == 3).all())
    assert int(torch.count_nonzero(out[:n].view(torch.int16).view(torch.int64))) <= len(some) * 64
    del keys, out
    torch.cuda.empty_cache()


# ---- the range of values ------------------------------------------------------------------------------------------------
def each_query(t, got, q, n0):
    """Every query by itself.  A share (weight times its value's scale) is rounded to an f16 (2^-11) and scores are off by 1e-5, together under 2^-10 of every share; the output is a bf16 (2^-8).
    A query's largest share is 2^5 or more (2^6 times a factor of 1/2 or more when its maximum was taken), and shares under 2^-14 are rounded by 2^-25: by 2^-30 of the largest, each.  (A
    column where the largest token's number is zero shows that: what the others leave there is small.)"""
    got = u.host(got).reshape(len(q), t.heads, -1)
    k, number, ks, vs = t.cache.host()
    k = k.astype(f64) * ks[..., None]
    for i in range(len(q)):
        p = n0 + i if np.ndim(n0) == 0 else n0[i]
        first = max(p // t.chunk * t.chunk if t.chunk else 0, p - t.window + 1 if t.window else 0)
        for h in range(t.heads):
            kvh = h // (t.heads // t.kv)
            s = k[kvh, 0, first:p + 1, :t.dim] @ q[i, h].astype(f64)
            e = np.exp(s - s.max())
            share, x = e / e.sum() * vs[kvh, first:p + 1], number[kvh, first:p + 1].astype(f64)
            want = share @ x
            off = np.abs(got[i, h] - want) - (2.0 ** -8 * np.abs(want) + 2.0 ** -10 * (share @ np.abs(x)) + 2.0 ** -30 * share.max() * np.abs(x).sum(0))
            assert off.max() <= 0, (p, h, off.argmax(), got[i, h, off.argmax()], want[off.argmax()])


def prompted_by_value(hip, t, n0, n):
    t.convolved = t.rows[:, :t.channels].astype(f64)
    if n0:
        t.fill(hip, 0, n0)
    _, q = t.fill(hip, n0, n)
    q = as_bf16(q) if t.f32 else q
    qh = u.host(q).reshape(n - n0, -1, t.dimp)[..., :t.dim]
    for split in (True, False):
        each_query(t, t.prompt(hip, q, n0, n, split), qh, n0)


@pytest.mark.parametrize("up", [-112, -100, -80, 60, 100])
@pytest.mark.parametrize("shape", [(4, 2, 64, 64), (4, 1, 128, 128), (2, 1, 200, 200)])
def test_values_all_small_or_all_large(hip, pkg, shape, up):
    """down to what a cache's scale can hold"""
    t = kv.Attention(pkg, 200, *shape, normed=False, f32=True)
    t.rows[:, t.channels - t.kv * t.vdimp:t.channels] *= np.float32(2.0 ** up)
    prompted_by_value(hip, t, 0, 200)
    t.check(t.step(hip, 199), t.want(t.q[199:], 199), STEP)


@pytest.mark.parametrize("up", [10, 24, 33, 50])
@pytest.mark.parametrize("where", ["later", "ahead of the window", "ahead of the chunk"])
@pytest.mark.parametrize("shape", [(4, 2, 64, 64), (4, 1, 128, 128), (2, 1, 200, 200)])
def test_a_large_value_that_a_query_does_not_see(hip, pkg, shape, where, up):
    """in the same tile of keys, and tiles away"""
    for n0, n in ((0, 250), (100, 330)):
        options = {"later": {}, "ahead of the window": dict(window=40), "ahead of the chunk": dict(chunk=90)}[where]
        t = kv.Attention(pkg, n, *shape, normed=False, f32=True, **options)
        at = t.channels - t.kv * t.vdimp
        for i, more in ((n0 + 45, 0), (n0 + 140, 8), (n - 1, 9)) if where == "later" else ((3, 0), (70, 3), (n0 + 33, 6), (n0 + 155, 9)):
            t.rows[i, at:t.channels] *= np.float32(2.0 ** (up + more))
        prompted_by_value(hip, t, n0, n)


@pytest.mark.parametrize("up", [10, 30, 60])
def test_a_large_value_of_no_weight(hip, pkg, up):
    """what a query sees and does not weigh leaves the others their bits"""
    n = 300
    t = kv.Attention(pkg, n, 4, 2, 64, 64, normed=False, f32=True)
    nq = 4 * t.dimp
    t.rows[:, :nq] = np.abs(t.rows[:, :nq])
    for i in (20, 130, 200):
        t.rows[i, nq:nq + 2 * t.dimp] = -40.0  # (scores of some -400)
        t.rows[i, nq + 2 * t.dimp:t.channels] *= np.float32(2.0 ** up)
    prompted_by_value(hip, t, 0, n)


@pytest.mark.parametrize("up", [10, 30, 60])
@pytest.mark.parametrize("shape", [(4, 2, 64, 64, 1), (4, 1, 64, 128, 2), (2, 1, 200, 200, 1)])
def test_a_large_value_of_no_weight_in_a_step(hip, pkg, shape, up):
    """shares of 2^-20 of the largest and more keep the 22 bits of a pair of f16 (2^-24 absolute where the largest is 2^5 at least: 2^-30 of it)"""
    n = 300
    t = kv.Attention(pkg, n, *shape, normed=False, f32=True)
    nq, nk = t.heads * t.maps * t.dimp, t.kv * t.maps * t.dimp
    t.rows[:, :nq] = np.abs(t.rows[:, :nq])
    for i in (20, 130, 200, 280):
        t.rows[i, nq:nq + nk] = np.where(np.arange(nk) % t.dimp < t.dim, -40.0, 0.0)  # (scores of some -400)
        t.rows[i, nq + nk:t.channels] *= np.float32(2.0 ** up)
    t.convolved = t.rows[:, :t.channels].astype(f64)
    t.fill(hip, 0, n - 1)
    q = t.rows[n - 1:, :nq].astype(f64).reshape(1, -1, t.dimp)[..., :t.dim] * t.keep[2][n - 1].item()
    t.check(t.step(hip, n - 1), t.want(q, n - 1), STEP)


@pytest.mark.parametrize("shape", [(4, 2, 24, 40, 2), (4, 2, 64, 64, 1), (6, 3, 96, 96, 1), (4, 2, 128, 128, 1), (2, 1, 200, 256, 2), (2, 2, 256, 256, 1)])
@pytest.mark.parametrize("rot", [0, 8, 24])
def test_a_step_writes_what_a_portion_of_one_writes(hip, pkg, shape, rot):
    """bit by bit where a norm's sum is exact (whole numbers) and has no order"""
    n = 60
    one, step = (kv.Attention(pkg, n, *shape, f32=True, rot=rot) for _ in range(2))
    for t in (one, step):
        nk = (t.heads + t.kv) * t.maps * t.dimp
        t.rows[:, :nk] = np.rint(t.rows[:, :nk] * 3)
        t.convolved = t.rows[:, :t.channels].astype(f64)
    for i in range(n):
        one.fill(hip, i, i + 1)
        step.step(hip, i)
    for name, a, b in zip(("keys", "values", "key scales", "value scales"), one.cache.host(), step.cache.host()):
        assert np.array_equal(a, b), (name, (a != b).mean())


@pytest.mark.parametrize("options", [dict(), dict(sink=True, gate="heads"), dict(gate="columns", window=700)])
@pytest.mark.parametrize("shape,n", [((20, 5, 128, 128, 1), 1), ((20, 5, 128, 128, 1), 129), ((20, 5, 128, 128, 1), 512), ((12, 3, 96, 96, 1), 1500), ((128, 128, 32, 32, 1), 640),
                                     ((128, 128, 32, 32, 1), 1100), ((128, 128, 24, 24, 1), 1500)])
def test_records_into_the_product_behind_them(hip, pkg, shape, n, options):
    """a step's records, joined ones and the empty ones behind them too (128 heads: two in one from 513 workgroups on, four from 1025), by gqa_project and, up to four, gqa_out: as by
    gqa_merge and a product in 64 bits"""
    t = kv.Attention(pkg, n, *shape, f32=True, **options)
    if n > 1:
        t.fill(hip, 0, n - 1)
    scratch = u.zeros_f32(hip.gqa_scratch_bytes(t.heads, 1, t.vdimp, 1) // 4)
    scratch.fill_(np.nan)
    out = t.step(hip, n - 1, scratch=scratch)
    t.check(out, t.want(t.q[n - 1:], n - 1), STEP)
    cols, rows = t.heads * t.vdimp, 70
    first = max(0, n - t.window) if t.window else 0
    records = (n - 1 - first // 128 * 128) // 128 + 1
    w = u.rounded(np.random.default_rng(n).standard_normal((rows, cols)) / np.sqrt(cols))
    row = u.dev_f32(t.rows[n - 1])  # (the gate that step took from a buffer of its own)
    t.gated(row)
    pos, want = u.dev(np.array([n - 1], np.int32)), w.astype(f64) @ u.host(out).reshape(-1).astype(f64)
    product = hip.gqa_project_dev, hip.gqa_out_dev
    for call, most in zip(product, (hip.gqa_project_records(t.attn, cols), hip.gqa_out_records(t.attn, cols))):
        assert most >= 4
        if records > most:
            continue
        y = u.zeros_f32(rows)
        call(t.attn, pos, records, scratch, u.dev_bf16(w), rows, cols, cols, y)
        assert u.rms_error(u.host(y), want) < 3e-6


# ---- every form of a prompt's launch --------------------------------------------------------------------------------------
# columns (keys, values), maps | groups, waves, stretches or not: heads, kv heads, keys, queries
FORMS = {
    (24, 64, 1): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (3, 1, 333, 111), (2, 4, False): (3, 1, 333, 111), (2, 4, True): (3, 1, 2000, 2000), (1, 8, False): (100, 5, 1000, 1000),
                  (1, 8, True): (6, 1, 2000, 2000)},
    (64, 100, 1): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (3, 1, 333, 111), (2, 4, False): (3, 1, 333, 111), (2, 4, True): (3, 1, 1600, 1600), (1, 8, False): (100, 5, 1000, 1000),
                   (1, 8, True): (32, 4, 2000, 500)},
    (100, 128, 1): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (3, 1, 333, 111), (2, 4, False): (3, 1, 333, 111), (2, 4, True): (3, 1, 1600, 1600), (1, 8, False): (100, 5, 1000, 1000),
                    (1, 8, True): (32, 4, 2000, 500)},
    (200, 256, 1): {(1, 4, False): (3, 1, 333, 111), (1, 4, True): (3, 1, 333, 111)},
    (24, 64, 2): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (1, 1, 333, 333), (2, 4, False): (1, 1, 333, 333), (2, 4, True): (2, 1, 1600, 1600), (1, 8, False): (100, 5, 500, 500),
                  (1, 8, True): (3, 1, 2000, 2000)},
    (64, 100, 2): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (1, 1, 333, 333), (2, 4, False): (1, 1, 333, 333), (2, 4, True): (2, 1, 1600, 1600), (1, 8, False): (100, 5, 500, 500),
                   (1, 8, True): (16, 4, 2000, 500)},
    (100, 128, 2): {(1, 4, False): (3, 1, 130, 130), (1, 4, True): (1, 1, 333, 333), (1, 8, False): (60, 3, 500, 500), (1, 8, True): (3, 1, 1600, 1600)},
    (200, 160, 2): {(1, 4, False): (3, 1, 60, 60), (1, 4, True): (3, 1, 333, 111)},
}
FORM_CASES = [(columns, form, shape, options) for columns, forms in FORMS.items() for form, shape in forms.items()
              for options in ([dict(rot=8)] if columns[2] == 2 else [dict(rot=8), dict(far=True), dict(gate="columns", sink=True), dict(far=True, gate="columns", rot=24)])]


@pytest.mark.parametrize("columns,form,shape,options", FORM_CASES)
def test_every_form_of_a_prompt(hip, pkg, columns, form, shape, options):
    """each way in which a launch can be shared out, with and without what stands in the instances of its own (penalty, gates by columns); a sample of the queries by definition"""
    heads, kvh, n, nq = shape
    t = kv.Attention(pkg, n, heads, kvh, *columns, fill=-128, scale=np.nan, **options)
    if n > nq:
        t.fill(hip, 0, n - nq)
    rows, q = t.fill(hip, n - nq, n)
    out = t.prompt(hip, q, n - nq, n, split=form[2])
    groups, waves, stretches = hip.kv8_prefill_last_form()
    assert (groups, waves, stretches > 1) == form
    some = np.unique(np.concatenate([np.linspace(0, nq - 1, 9).astype(int), [min(nq - 1, 31), min(nq - 1, 64), nq - 2]]))
    held, qh = t.cache.held(), u.host(q).reshape(nq, -1, t.dimp)[..., :t.dim]
    want = np.concatenate([t.want(qh[i:i + 1], n - nq + i, held) for i in some])
    t.check(u.dev_f32(u.host(out)[some]), want, *PROMPT)


@pytest.mark.parametrize("columns,form,shape", [(columns, form, shape) for columns, forms in FORMS.items() if columns[2] == 1 for form, shape in forms.items()])
def test_every_form_beside_large_values(hip, pkg, columns, form, shape):
    """large values that the queries ahead of them do not see, in every stretch and group"""
    heads, kvh, n, nq = shape
    t = kv.Attention(pkg, n, heads, kvh, *columns, normed=False, f32=True)
    first = t.channels - t.kv * t.vdimp
    for i, up in zip(np.linspace(n - nq, n - 1, 7).astype(int), (0, 20, 26, 31, 37, 41, 60)):
        t.rows[i, first:t.channels] *= np.float32(2.0 ** up)
    if n > nq:
        t.fill(hip, 0, n - nq)
    _, q = t.fill(hip, n - nq, n)
    q = as_bf16(q)
    out = t.prompt(hip, q, n - nq, n, split=form[2])
    groups, waves, stretches = hip.kv8_prefill_last_form()
    assert (groups, waves, stretches > 1) == form
    some = np.unique(np.concatenate([np.linspace(0, nq - 2, 9).astype(int), np.linspace(0, nq - 1, 7).astype(int)[1:] - 1]))
    each_query(t, u.dev_f32(u.host(out)[some]), u.host(q).reshape(nq, -1, t.dimp)[some][..., :t.dim], n - nq + some)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("shape,n0,n", [((64, 64, 32, 32, 1), 5, 1100), ((30, 30, 24, 40, 2), 32, 2300)])
def test_many_tokens_of_many_heads_of_either_type(hip, pkg, shape, n0, n, f32):
    """values by pieces of 32 positions, as test_many_tokens_of_many_heads"""
    test_written_bit_by_bit(hip, pkg, shape, n0, n, f32)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("taps", [1, 3, 5])
@pytest.mark.parametrize("shape,n0,n", [((40, 40, 64, 64, 1), 13, 1700), ((32, 32, 24, 40, 2), 45, 2100), ((16, 16, 100, 128, 1), 70, 4200), ((6, 2, 200, 256, 1), 33, 300)])
def test_convolutions_of_many_tokens(hip, pkg, shape, n0, n, taps, f32):
    """pieces of 32 positions and of eight; a second portion that begins inside a tile, with the first one's last rows in the ring"""
    t = kv.Attention(pkg, n0 + n, *shape, f32=f32, taps=taps)
    for a, b in ((0, n0), (n0, n0 + n)):
        _, q = t.fill(hip, a, b)
        got = u.host(q).reshape(b - a, -1, t.dimp)
        assert u.rms_error(got[..., :t.dim], t.q[a:b]) < (3e-6 if f32 else 2.0 ** -8)
    k, v, ks, vs = t.cache.host()
    for got, scales, x in ((k, ks, t.k), (v, vs, t.v)):
        got, scales = got[..., :n0 + n, :].astype(np.float32), scales[..., :n0 + n]
        largest = np.abs(x).max(-1)
        assert np.abs(scales * 127 / largest - 1).max() < 1e-5
        assert (np.abs(got * scales[..., None] - x) <= scales[..., None] * 0.5 + 1e-5 * largest[..., None]).all()


@pytest.mark.parametrize("up", [95, -95])
def test_queries_and_keys_at_the_ends_of_their_range(hip, pkg, up):
    """queries of some 2^-98 and keys of some 2^98, and the other way round"""
    test_queries_and_keys_of_opposite_size(hip, pkg, up)
