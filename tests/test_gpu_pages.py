"""The 8-bit cache of pages: appends, the row step, attention over a ragged batch,
reading back and refusals, against the block format restated in NumPy and against
64-bit attention."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24  # half a step of FP32
BLOCK = 16


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def int32(values):
    return to_dev(np.asarray(values, dtype=np.int32))


def starts(counts):
    return int32(np.concatenate([[0], np.cumsum(counts)]))


def decoded_block(x):
    """What a block of rows [n][heads][64] (n up to 16) holds, every step in FP32."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        scale = (np.abs(x).max(axis=(0, 2)) / F32(127)).astype(F32)
        small = scale < F32(2.0 ** -126)
        inverse = np.where(small, F32(0), (F32(1) / scale).astype(F32)).astype(F32)
        codes = np.rint((x * inverse[None, :, None]).astype(F32)) + F32(0)  # integers: no negative zero
        out = (codes * np.where(small, F32(0), scale)[None, :, None]).astype(F32)
    out[:, ~np.isfinite(x).all(axis=(0, 2))] = np.nan
    return out


def decoded(x):
    """What the cache holds of a sequence's rows [n][heads][64]."""
    return np.concatenate([decoded_block(x[b:b + BLOCK]) for b in range(0, len(x), BLOCK)]) if len(x) else x


def make(fh, totals, page=64, heads=16, kv_heads=8, key_heads=None, seed=0, spare=3, ctx=None, seq_pages=None):
    """A cache whose sequences hold `totals` positions in pages of a random order."""
    rng = np.random.Generator(np.random.PCG64(seed))
    counts = [max(1, -(-t // page)) for t in totals]
    n_pages = sum(counts) + spare
    kv = fh.KvPages(n_pages, page, len(totals), seq_pages or max(counts), heads, kv_heads, key_heads=key_heads, ctx=ctx)
    ids = rng.permutation(n_pages)
    at = 0
    for i, n in enumerate(counts):
        kv.map(i, 0, ids[at:at + n])
        at += n
    return kv


def rows_of(counts, heads, seed, scale=1.0):
    return [gen.normal((n, heads, 64), scale, seed + 31 * i) for i, n in enumerate(counts)]


def cat(rows):
    return to_dev(np.concatenate(rows).astype(F32))


HEADS = [(16, 8, 8), (16, 8, 16), (4, 4, 4), (6, 1, 1), (6, 3, 6)]


@pytest.mark.parametrize("heads,kv_heads,key_heads", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_append_holds_the_blocks(fh, heads, kv_heads, key_heads, page):
    totals = [1, 15, 16, 17, 0, 64, 65, 100, 200]
    kv = make(fh, totals, page, heads, kv_heads, key_heads, seed=page)
    k, v = rows_of(totals, key_heads, 1), rows_of(totals, kv_heads, 1000)
    lens, row_start = int32([0] * len(totals)), starts(totals)
    kv.append(cat(k), cat(v), lens, row_start=row_start)
    gk, gv = kv.dequantize(sum(totals), lens, row_start=row_start)
    assert_bitwise(host(gk), np.concatenate([decoded(x) for x in k]), "keys")
    assert_bitwise(host(gv), np.concatenate([decoded(x) for x in v]), "values")
    assert kv.refused() == []


@pytest.mark.parametrize("page", [16, 32])
def test_appends_of_any_size_hold_the_same(fh, page):
    # The same rows in one call, and in calls of 1 to 40 rows each.
    totals = [90, 37, 130]
    k, v = rows_of(totals, 16, 3), rows_of(totals, 8, 5)
    whole, parts = (make(fh, totals, page, key_heads=16, seed=s) for s in (1, 2))
    zero = int32([0, 0, 0])
    whole.append(cat(k), cat(v), zero, row_start=starts(totals))
    rng = np.random.Generator(np.random.PCG64(7))
    at = [0, 0, 0]
    while at != totals:
        n = [min(t - a, int(rng.integers(0, rng.choice([2, 6, 41])))) for t, a in zip(totals, at)]
        if sum(n):
            parts.append(cat([x[a:a + m] for x, a, m in zip(k, at, n)]), cat([x[a:a + m] for x, a, m in zip(v, at, n)]),
                         int32(at), row_start=starts(n))
        at = [a + m for a, m in zip(at, n)]
        held = [host(x) for x in parts.dequantize(sum(at), zero, row_start=starts(at))] if sum(at) else None
        if held:
            assert_bitwise(held[0], np.concatenate([decoded(x[:a]) for x, a in zip(k, at)]), f"keys at {at}")
            assert_bitwise(held[1], np.concatenate([decoded(x[:a]) for x, a in zip(v, at)]), f"values at {at}")
    for got, want in zip(parts.dequantize(sum(totals), zero, row_start=starts(totals)),
                         whole.dequantize(sum(totals), zero, row_start=starts(totals))):
        assert_bitwise(host(got), host(want))


@pytest.mark.parametrize("length,back", [(40, 5), (33, 2), (33, 1), (48, 16), (50, 16), (17, 17)])
def test_positions_taken_back(fh, length, back):
    # Rejected drafts: up to 16 positions leave no trace.
    kv = make(fh, [80])
    k, v = rows_of([length], 8, 11, 2.0)[0], rows_of([length], 8, 13)[0]
    k[length - back:] *= F32(9.0)
    new_k, new_v = rows_of([7], 8, 17)[0], rows_of([7], 8, 19)[0]
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=starts([length]))
    kept = length - back
    kv.append(to_dev(new_k), to_dev(new_v), int32([kept]), row_start=starts([7]))
    gk, gv = kv.dequantize(kept + 7, int32([0]), row_start=starts([kept + 7]))
    assert_bitwise(host(gk), decoded(np.concatenate([k[:kept], new_k])))
    assert_bitwise(host(gv), decoded(np.concatenate([v[:kept], new_v])))


@pytest.mark.parametrize("kept", [3, 21])
def test_blocks_that_are_not_in_fp32_go_on_from_their_codes(fh, kept):
    # Further back than the FP32 blocks reach, and a sequence that goes on in pages it was given.
    length = 60
    k, v = rows_of([length], 8, 23)[0], rows_of([length], 8, 29)[0]
    new_k, new_v = rows_of([2], 8, 31, 3.0)[0], rows_of([2], 8, 37)[0]
    want = []
    for old, new in ((k, new_k), (v, new_v)):
        base = kept // BLOCK * BLOCK
        earlier = decoded(old)
        want.append(np.concatenate([earlier[:base], decoded_block(np.concatenate([earlier[base:kept], new]))]))
    for given in (False, True):
        kv = fh.KvPages(8, 16, 2, 4)
        kv.map(0, 0, [5, 2, 7, 0])
        kv.append(to_dev(k), to_dev(v), int32([0]), row_start=starts([length]))
        seq = 0
        if given:
            seq = 1
            # An own block that the given pages replace.
            kv.map(1, 0, [1, 3])
            kv.append(to_dev(new_k[:1]), to_dev(new_v[:1]), int32([-1, kept]), row_start=int32([0, 0, 1]))
            kv.map(1, 0, [5, 2, 7, 0])
        lens = int32([-1, kept] if given else [kept, -1])
        kv.append(to_dev(new_k), to_dev(new_v), lens, row_start=int32([0, 0, 2] if given else [0, 2, 2]))
        n = kept + 2
        gk, gv = kv.dequantize(n, int32([-1, 0] if given else [0, -1]), row_start=int32([0, 0, n] if given else [0, n, n]))
        assert_bitwise(host(gk), want[0], f"given {given}")
        assert_bitwise(host(gv), want[1], f"given {given}")


@pytest.mark.parametrize("heads,kv_heads,key_heads", HEADS)
def test_row_step_is_the_two_calls(fh, heads, kv_heads, key_heads):
    # Bitwise qkv_rows, then append of its keys and values.
    import torch

    counts, before = [1, 0, 20, 5, 70], [3, 9, 14, 32, 0]
    rows = sum(counts)
    totals = [a + b for a, b in zip(counts, before)]
    qkv = to_dev(gen.normal((rows, (heads + 2 * kv_heads) * 64), 1.0, 41))
    angle = gen.uniform((rows, heads, 32), -9.0, 9.0, 43)
    rope = to_dev(np.stack([np.cos(angle), np.sin(angle)], axis=-1).astype(F32))
    one, two = (make(fh, totals, 32, heads, kv_heads, key_heads, seed=s) for s in (1, 2))
    k0, v0 = cat(rows_of(before, key_heads, 47)), cat(rows_of(before, kv_heads, 53))
    zero, lens, row_start = int32([0] * 5), int32(before), starts(counts)
    for kv in (one, two):
        kv.append(k0, v0, zero, row_start=starts(before))
    q = one.qkv_rows(qkv, rope, lens, row_start=row_start)
    v = torch.empty((rows, kv_heads, 64), device="cuda:0")
    if key_heads == heads:
        k = torch.empty((rows, heads, 64), device="cuda:0")
        want = fh.qkv_rows(qkv, rows, rope, heads, kv_heads, rows, prefix_k=k, v=v)
    else:
        k = torch.empty((rows, kv_heads, 64), device="cuda:0")
        want = fh.qkv_rows(qkv, rows, rope, heads, kv_heads, 0, generated_k=k, v=v)
    two.append(k, v, lens, row_start=row_start)
    assert_bitwise(host(q), host(want), "queries")
    for a, b in zip(one.dequantize(sum(totals), zero, row_start=starts(totals)),
                    two.dequantize(sum(totals), zero, row_start=starts(totals))):
        assert_bitwise(host(a), host(b))


@pytest.mark.parametrize("heads,kv_heads,key_heads", HEADS)
@pytest.mark.parametrize("counts,before", [([1500], [5]), ([1400, 0, 2, 3000], [0, 40, 33, 17])])
def test_long_prompts_are_their_parts(fh, heads, kv_heads, key_heads, counts, before):
    # A thousand rows a sequence and more in one call, or as many calls as it takes of up to 300.
    totals = [a + b for a, b in zip(counts, before)]
    rows, n = sum(counts), len(counts)
    qkv = to_dev(gen.normal((rows, (heads + 2 * kv_heads) * 64), 1.0, 61))
    angle = gen.uniform((rows, heads, 32), -9.0, 9.0, 62)
    rope = to_dev(np.stack([np.cos(angle), np.sin(angle)], axis=-1).astype(F32))
    one, two = (make(fh, totals, 64, heads, kv_heads, key_heads, seed=s) for s in (1, 2))
    k0, v0 = cat(rows_of(before, key_heads, 63)), cat(rows_of(before, kv_heads, 64))
    zero = int32([0] * n)
    for kv in (one, two):
        kv.append(k0, v0, zero, row_start=starts(before))
    q = host(one.qkv_rows(qkv, rope, int32(before), row_start=starts(counts)))
    first = np.cumsum([0] + counts)
    for i in range(n):
        for at in range(0, counts[i], 300):
            size = min(300, counts[i] - at)
            lens, row_start = [-1] * n, [0] * (i + 1) + [size] * (n - i)
            lens[i] = before[i] + at
            here = slice(first[i] + at, first[i] + at + size)
            part = two.qkv_rows(qkv[here].contiguous(), rope[here].contiguous(), int32(lens), row_start=int32(row_start))
            assert_bitwise(q[here], host(part), f"queries of sequence {i} from {at}")
    for a, b in zip(one.dequantize(sum(totals), zero, row_start=starts(totals)),
                    two.dequantize(sum(totals), zero, row_start=starts(totals))):
        assert_bitwise(host(a), host(b))
    assert one.refused() == [] and two.refused() == []


def attention64(q, k, v, first, sinks):
    """64-bit attention of rows [n][H][64] at positions first.. over decoded keys and
    values, and how far FP32's may be from it.

    A score is off by the query's step (2^-22 of the row's largest element) times the
    key, and a few roundings of itself and of its exponent; a weight by the
    exponential of twice that (its own and the maximum's). A weighted value passes up
    to 32 roundings in its matrix product, one for each 32 keys and each 64 keys of
    its part, and some 80 where parts meet. It enters its product as an integer of
    2^-30 of a power of two that is at most twice the largest block scale of its
    run: off by half of that, 2^-30 of the largest value, for each key of a run (4,096
    at most), relative to the run's largest weight, which is part of its sum: so over
    all runs 2^-30 of the largest value for each key of the longest."""
    n, heads, _ = q.shape
    out, bound = np.empty(q.shape), np.empty(q.shape)
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for h in range(heads):
        kh, vh = k[:, h * k.shape[1] // heads], v[:, h * v.shape[1] // heads]
        for r in range(n):
            seen = first + r + 1
            s = kh[:seen] @ q[r, h] / 8.0
            w = np.exp(s - s.max())
            total = w.sum()
            sink = 1.0 if sinks is None else 1.0 / (1.0 + np.exp(sinks[h] - s.max() - np.log(total)))
            out[r, h] = w @ vh[:seen] / total * sink
            off = 4 * EPS * np.abs(q[r, h]).max() * np.abs(kh[:seen]).sum(axis=1).max() / 8 + EPS * (8 * np.abs(s).max() + 16)
            size = w @ np.abs(vh[:seen]) / total * sink
            least = min(seen, 4096) * 2.0 ** -30 * np.abs(vh[:seen]).max() * sink
            bound[r, h] = size * (2.2 * off + EPS * (seen / 20 + 112)) + least + 1e-40
    return out, bound


def check(got, want, bound, label=""):
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= bound).all(), f"{label}: {np.max(off / bound)} times what is allowed, off by {off.max()}"


def attend(fh, totals, counts, page=64, heads=16, kv_heads=8, key_heads=None, sinks=True, seed=0, scale=1.0, max_len=None):
    kv = make(fh, totals, page, heads, kv_heads, key_heads, seed=seed)
    k, v = rows_of(totals, kv.key_heads, seed + 1, scale), rows_of(totals, kv_heads, seed + 2)
    zero = int32([0] * len(totals))
    kv.append(cat(k), cat(v), zero, row_start=starts(totals))
    q = rows_of(counts, heads, seed + 3)
    s = gen.normal((heads,), 1.0, seed + 4) if sinks else None
    before = [t - c for t, c in zip(totals, counts)]
    got = host(kv.attention(cat(q), int32(before), max_len or max(totals), row_start=starts(counts),
                            sinks=None if s is None else to_dev(s)))
    assert kv.refused() == []
    at = 0
    for i, (b, c) in enumerate(zip(before, counts)):
        if c:
            check(got[at:at + c], *attention64(q[i], decoded(k[i]), decoded(v[i]), b, s),
                  f"sequence {i}: {c} rows after {b}")
        at += c


@pytest.mark.parametrize("heads,kv_heads,key_heads", HEADS)
@pytest.mark.parametrize("page", [16, 128])
def test_attention_of_a_ragged_batch(fh, heads, kv_heads, key_heads, page):
    attend(fh, [1, 2, 15, 16, 17, 63, 64, 65, 100, 129, 300], [1, 2, 3, 8, 1, 4, 5, 6, 7, 0, 8], page, heads, kv_heads,
           key_heads, seed=page + heads)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 7, 8])
def test_attention_of_every_row_count(fh, rows):
    attend(fh, [900, 70], [rows, 1], 32, seed=rows, sinks=rows % 2 == 0)


@pytest.mark.parametrize("heads,kv_heads,key_heads,total,rows", [(16, 8, 8, 5000, 3), (16, 8, 16, 2600, 8),
                                                                (32, 1, 1, 700, 8), (2, 1, 2, 40000, 1)])
def test_attention_over_long_caches(fh, heads, kv_heads, key_heads, total, rows):
    attend(fh, [total, total // 3], [rows, min(rows, 2)], 64, heads, kv_heads, key_heads, seed=total)


def test_attention_with_peaked_scores_and_a_loose_bound(fh):
    # Large keys: a few positions take all the weight. max_len far above the lengths.
    attend(fh, [500, 40], [5, 8], 64, seed=61, scale=12.0)
    kv_len = 64 * 40
    kv = fh.KvPages(64, 64, 2, 40)
    kv.map(0, 0, list(range(40)))
    kv.map(1, 0, [50])
    k, v, q = gen.normal((100, 8, 64), 1.0, 67), gen.normal((100, 8, 64), 1.0, 71), gen.normal((2, 16, 64), 1.0, 73)
    kv.append(to_dev(k), to_dev(v), int32([0, 0]), row_start=int32([0, 70, 100]))
    got = host(kv.attention(to_dev(q), int32([69, 29]), kv_len))
    for i, (lo, hi) in enumerate(((0, 70), (70, 100))):
        check(got[i:i + 1], *attention64(q[i:i + 1], decoded(k[lo:hi]), decoded(v[lo:hi]), hi - lo - 1, None), f"{i}")


def test_values_of_every_magnitude(fh):
    # Blocks with scales far apart, zero blocks, blocks below the smallest scale.
    total = 130
    k, v = gen.normal((total, 8, 64), 1.0, 79), gen.normal((total, 8, 64), 1.0, 83)
    v[:16] *= F32(1e-8)
    v[16:32] *= F32(1e6)
    v[32:48] = 0
    k[48:64] = 0
    k[64:80] *= F32(1e-30)
    v[64:80] *= F32(1e-38)
    v[80:96] *= F32(1e-40)
    kv = make(fh, [total])
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=starts([total]))
    gk, gv = (host(x) for x in kv.dequantize(total, int32([0]), row_start=starts([total])))
    assert_bitwise(gk, decoded(k))
    assert_bitwise(gv, decoded(v))
    q = gen.normal((4, 16, 64), 1.0, 89)
    got = host(kv.attention(to_dev(q), int32([total - 4]), total, row_start=starts([4])))
    want, bound = attention64(q, gk, gv, total - 4, None)
    check(got, want, bound)


def test_huge_and_tiny_queries(fh):
    k, v = gen.normal((50, 8, 64), 1e-20, 97), gen.normal((50, 8, 64), 1.0, 101)
    kv = make(fh, [50])
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=starts([50]))
    q = gen.normal((3, 16, 64), 1.0, 103) * np.array([1e20, 1e-30, 0.0], dtype=F32)[:, None, None]
    got = host(kv.attention(to_dev(q.astype(F32)), int32([47]), 50, row_start=starts([3])))
    check(got, *attention64(q.astype(F32), decoded(k), decoded(v), 47, None))


def test_non_finite_rows(fh):
    # Position 20 of key head 2 and position 37 of value head 5 poison their blocks: rows
    # that see them are NaN in those heads, earlier rows and other heads keep their values.
    # Written again, the blocks are what they would have been.
    total = 40
    k, v = gen.normal((total, 8, 64), 1.0, 107), gen.normal((total, 8, 64), 1.0, 109)
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[36, 2, 7] = np.inf
    bad_v[37, 5, 0] = np.nan
    q = gen.normal((8, 16, 64), 1.0, 113)
    kv = make(fh, [total])
    kv.append(to_dev(bad_k), to_dev(bad_v), int32([0]), row_start=starts([total]))
    gk, gv = (host(x) for x in kv.dequantize(total, int32([0]), row_start=starts([total])))
    assert_bitwise(gk, decoded(bad_k))
    assert_bitwise(gv, decoded(bad_v))
    got = host(kv.attention(to_dev(q), int32([28]), total, row_start=starts([8])))  # rows at 28 .. 35
    want, bound = attention64(q, decoded(k), decoded(v), 28, None)
    nan = np.isnan(got).all(axis=2)
    poisoned = np.zeros((8, 16), bool)
    poisoned[4:, [4, 5, 10, 11]] = True  # from position 32 on
    assert np.array_equal(nan, poisoned)
    got2, want2, bound2 = got[:4], want[:4], bound[:4]
    check(got2, want2, bound2)
    fine = ~poisoned
    fine[4:] &= np.ones(16, bool)
    later = [h for h in range(16) if h not in (4, 5, 10, 11)]
    wk, wv = decoded(bad_k), decoded(bad_v)
    want, bound = attention64(q[:, later], wk[:, [h // 2 for h in later]], wv[:, [h // 2 for h in later]], 28, None)
    check(got[:, later], want, bound)
    kv.append(to_dev(k[36:]), to_dev(v[36:]), int32([36]), row_start=starts([4]))
    gk, gv = (host(x) for x in kv.dequantize(total, int32([0]), row_start=starts([total])))
    assert_bitwise(gk, decoded(k))
    assert_bitwise(gv, decoded(v))


def test_non_finite_queries(fh):
    k, v, q = gen.normal((30, 8, 64), 1.0, 127), gen.normal((30, 8, 64), 1.0, 131), gen.normal((3, 16, 64), 1.0, 137)
    kv = make(fh, [30])
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=starts([30]))
    want, bound = attention64(q, decoded(k), decoded(v), 27, None)
    q[1, 3, 9], q[2, 8, 63] = np.nan, np.inf
    got = host(kv.attention(to_dev(q), int32([27]), 30, row_start=starts([3])))
    nan = np.zeros((3, 16), bool)
    nan[1, 3] = nan[2, 8] = True
    assert np.array_equal(np.isnan(got).all(axis=2), nan) and np.array_equal(np.isnan(got).any(axis=2), nan)
    check(got[~nan], want[~nan], bound[~nan])


def test_refused_and_idle_sequences(fh):
    import torch

    # 0 idle, 1 fine, 2 past its pages, 3 a page missing, 4 nine rows, 5 longer than max_len, 6 rows out
    # of range, 7 fine; a row before the first sequence and one behind the last.
    page = 16
    kv = fh.KvPages(40, page, 8, 4)
    for i in range(8):
        kv.map(i, 0, [4 * i, 4 * i + 1, -1 if i == 3 else 4 * i + 2, 4 * i + 3])
    counts = [1, 2, 3, 2, 9, 1, 1, 2]
    before = [-1, 10, 62, 31, 5, 60, 8, 20]
    row_start = np.concatenate([[1], 1 + np.cumsum(counts)]).astype(np.int32)
    rows = int(row_start[-1]) + 1
    first = row_start[:-1].copy()
    k0, v0 = rows_of([60] * 8, 8, 139), rows_of([60] * 8, 8, 149)
    full = [0, 10, 60, 32, 60, 60, 60, 20]
    kv.append(cat([x[:n] for x, n in zip(k0, full)]), cat([x[:n] for x, n in zip(v0, full)]), int32([0] * 8),
              row_start=starts(full))
    assert kv.refused() == []
    k, v, q = gen.normal((rows, 8, 64), 1.0, 151), gen.normal((rows, 8, 64), 1.0, 157), gen.normal((rows, 16, 64), 1.0, 163)
    row_start[7] = rows + 5  # sequence 6 ends, and 7 begins, past the rows
    row_start[8] = rows + 5
    kv.append(to_dev(k), to_dev(v), int32(before), row_start=int32(row_start))
    assert kv.refused() == [2, 3, 6, 7]
    assert kv.refused() == []
    row_start = np.concatenate([[1], 1 + np.cumsum(counts)]).astype(np.int32)
    kv.append(to_dev(k[first[7]:first[7] + 2]), to_dev(v[first[7]:first[7] + 2]), int32([-1] * 7 + [20]),
              row_start=int32([0] * 8 + [2]))
    out = torch.full((rows, 16, 64), 123.0, device="cuda:0")
    kv.attention(to_dev(q), int32(before), 56, row_start=int32(row_start), out=out)
    assert kv.refused() == [2, 3, 4, 5]
    got = host(out)
    untouched = [0, 1, rows - 1]  # before the first, the idle one's, behind the last
    assert (got[untouched] == 123.0).all()
    for i in (2, 4, 5):
        assert np.isnan(got[first[i]:first[i] + counts[i]]).all(), i
    a = first[3]
    assert np.isnan(got[a + 1]).all()  # its position 32 has no page
    want, bound = attention64(q[a:a + 1], decoded(np.concatenate([k0[3][:31], k[a:a + 1]])),
                              decoded(np.concatenate([v0[3][:31], v[a:a + 1]])), 31, None)
    check(got[a:a + 1], want, bound, "the row before the missing page")
    for i in (1, 6, 7):
        a, n, b = first[i], counts[i], before[i]
        if i == 6:
            kk, vv = decoded(k0[i]), decoded(v0[i])  # its append was refused
        else:
            kk = decoded(np.concatenate([k0[i][:b], k[a:a + n]]))
            vv = decoded(np.concatenate([v0[i][:b], v[a:a + n]]))
        check(got[a:a + n], *attention64(q[a:a + n], kk, vv, b, None), f"sequence {i}")
    gk, gv = kv.dequantize(2, int32([-1, -1, -1, 31, -1, -1, -1, -1]), row_start=int32([0, 0, 0, 0, 2, 2, 2, 2, 2]))
    assert np.isnan(host(gk)[1]).all() and np.isnan(host(gv)[1]).all() and np.isfinite(host(gk)[0]).all()
    assert kv.refused() == [3]
    # Rows that overlap the sequence's before it.
    kv.append(to_dev(k[:4]), to_dev(v[:4]), int32([0, 0, 0, 0, 0, 0, 0, 0]), row_start=int32([0, 4, 2, 4, 4, 4, 4, 4, 4]))
    assert kv.refused() == [1, 2]


def test_queries_of_idle_and_refused_sequences_stay(fh):
    import torch

    kv = make(fh, [20, 20, 20, 20])
    qkv = to_dev(gen.normal((6, 32 * 64), 1.0, 167))
    rope = to_dev(np.tile(np.array([1, 0], F32), (6, 16, 32, 1)))
    q = torch.full((6, 16, 64), 5.0, device="cuda:0")
    kv.qkv_rows(qkv, rope, int32([0, -1, 64, 3]), row_start=int32([1, 2, 3, 4, 5]), q=q)
    got = host(q)
    assert (got[[0, 2, 3, 5]] == 5.0).all() and (got[[1, 4]] != 5.0).all()
    assert kv.refused() == [2]


def test_many_sequences_of_uneven_rows(fh):
    # More sequences than a wave looks through at once.
    rng = np.random.Generator(np.random.PCG64(173))
    counts = [int(rng.integers(0, 40)) for _ in range(150)]
    kv = make(fh, counts, 16, 2, 1, 2, seed=5)
    k, v = rows_of(counts, 2, 179), rows_of(counts, 1, 181)
    zero = int32([0] * 150)
    kv.append(cat(k), cat(v), zero, row_start=starts(counts))
    gk, gv = kv.dequantize(sum(counts), zero, row_start=starts(counts))
    assert_bitwise(host(gk), np.concatenate([decoded(x) for x in k]))
    assert_bitwise(host(gv), np.concatenate([decoded(x) for x in v]))
    last = [min(c, 8) for c in counts]
    q = rows_of(last, 2, 191)
    got = host(kv.attention(cat(q), int32([c - n for c, n in zip(counts, last)]), 40, row_start=starts(last)))
    at = 0
    for i, n in enumerate(last):
        if n:
            check(got[at:at + n], *attention64(q[i], decoded(k[i]), decoded(v[i]), counts[i] - n, None), f"sequence {i}")
        at += n


def test_offsets_past_32_bits(fh):
    # 2.4 GB of key codes: the last pages' offsets do not fit 32 bits.
    page, heads = 4096, 16
    n_pages = 580
    kv = fh.KvPages(n_pages, page, 2, 2, heads, 8, key_heads=16)
    assert kv.device_bytes() > 3 * 2 ** 30
    kv.map(0, 0, [n_pages - 1, 0])
    kv.map(1, 0, [n_pages - 2])
    totals = [4100, 50]
    k, v, q = rows_of(totals, 16, 193), rows_of(totals, 8, 197), rows_of([2, 1], heads, 199)
    kv.append(cat(k), cat(v), int32([0, 0]), row_start=starts(totals))
    gk, gv = kv.dequantize(sum(totals), int32([0, 0]), row_start=starts(totals))
    assert_bitwise(host(gk), np.concatenate([decoded(x) for x in k]))
    assert_bitwise(host(gv), np.concatenate([decoded(x) for x in v]))
    got = host(kv.attention(cat(q), int32([4098, 49]), 4100, row_start=starts([2, 1])))
    check(got[:2], *attention64(q[0], decoded(k[0]), decoded(v[0]), 4098, None))
    check(got[2:], *attention64(q[1], decoded(k[1]), decoded(v[1]), 49, None))


def test_shared_pages(fh):
    # Two sequences read the full pages of a common prompt and write their own.
    page = 32
    kv = fh.KvPages(5, page, 2, 3)
    kv.map(0, 0, [3, 1, 4])
    prompt_k, prompt_v = gen.normal((64, 8, 64), 1.0, 211), gen.normal((64, 8, 64), 1.0, 223)
    kv.append(to_dev(prompt_k), to_dev(prompt_v), int32([0, -1]), row_start=int32([0, 64, 64]))
    kv.map(1, 0, [3, 1, 0])
    k, v, q = gen.normal((10, 8, 64), 1.0, 227), gen.normal((10, 8, 64), 1.0, 229), gen.normal((10, 16, 64), 1.0, 233)
    lens, row_start = int32([64, 64]), int32([0, 4, 10])
    kv.append(to_dev(k), to_dev(v), lens, row_start=row_start)
    got = host(kv.attention(to_dev(q), lens, 70, row_start=row_start))
    for lo, hi in ((0, 4), (4, 10)):
        kk = decoded(np.concatenate([prompt_k, k[lo:hi]]))
        vv = decoded(np.concatenate([prompt_v, v[lo:hi]]))
        check(got[lo:hi], *attention64(q[lo:hi], kk, vv, 64, None))


def test_captured_steps_advance_on_the_device(fh):
    import torch

    # One graph decodes step after step: lengths are advanced by the graph itself.
    n_seqs, steps = 3, 40
    totals = [60 + steps, 7 + steps, 16 + steps]
    before = [60, 7, 16]
    ctx = fh.Context(0)
    one, two = make(fh, totals, 16, seed=1, ctx=ctx), make(fh, totals, 16, seed=2, ctx=ctx)
    k0, v0 = cat(rows_of(before, 8, 239)), cat(rows_of(before, 8, 241))
    zero = int32([0] * n_seqs)
    for kv in (one, two):
        kv.append(k0, v0, zero, row_start=starts(before))
    qkv = torch.zeros(n_seqs, 32 * 64, device="cuda:0")
    rope = to_dev(np.tile(np.array([0.6, 0.8], F32), (n_seqs, 16, 32, 1)))
    lens, q, out = int32(before), torch.zeros(n_seqs, 16, 64, device="cuda:0"), torch.zeros(n_seqs, 16, 64, device="cuda:0")
    most = max(totals)
    sinks = to_dev(gen.normal((16,), 1.0, 251))
    two.attention(q, int32(before), most, sinks=sinks)  # the scratch grows uncaptured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        one.qkv_rows(qkv, rope, lens, q=q)
        one.attention(q, lens, most, sinks=sinks, out=out)
        lens.add_(1)
    ctx.use_stream(torch.cuda.current_stream())
    for step in range(steps):
        qkv.copy_(to_dev(gen.normal((n_seqs, 32 * 64), 1.0, 257 + step)))
        graph.replay()
        torch.cuda.synchronize()
        got = host(out)
        at = int32([b + step for b in before])
        want = two.attention(two.qkv_rows(qkv, rope, at), at, most, sinks=sinks)
        assert_bitwise(got, host(want), f"step {step}")
    assert host(lens).tolist() == totals
    assert one.refused() == two.refused() == []


def test_two_streams_and_contexts(fh):
    import torch

    ctxs = [fh.Context(0), fh.Context(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got, wants = [], []
    for i, (ctx, stream) in enumerate(zip(ctxs, streams)):
        stream.wait_stream(torch.cuda.current_stream())
        ctx.use_stream(stream)
        total = 700 + 100 * i
        kv = make(fh, [total], seed=i, ctx=ctx)
        k, v, q = gen.normal((total, 8, 64), 1.0, 263 + i), gen.normal((total, 8, 64), 1.0, 269 + i), gen.normal((4, 16, 64), 1.0, 271 + i)
        args = [to_dev(k), to_dev(v), to_dev(q), int32([0]), starts([total]), int32([total - 4]), starts([4])]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            kv.append(args[0], args[1], args[3], row_start=args[4])
            got.append((kv.attention(args[2], args[5], total, row_start=args[6]), kv, args))
        wants.append(attention64(q, decoded(k), decoded(v), total - 4, None))
    torch.cuda.synchronize()
    for (out, _, _), (want, bound) in zip(got, wants):
        check(host(out), want, bound)


def test_empty_calls(fh):
    import torch

    kv = make(fh, [16])
    none = torch.empty(0, 8, 64, device="cuda:0")
    kv.append(none, none, int32([0]), row_start=int32([0, 0]))
    out = kv.attention(torch.empty(0, 16, 64, device="cuda:0"), int32([0]), 16, row_start=int32([0, 0]))
    assert out.shape == (0, 16, 64)
    k, v = kv.dequantize(0, int32([0]), row_start=int32([0, 0]))
    assert k.shape == v.shape == (0, 8, 64)
    kv.map(0, 1, [])
    assert kv.refused() == []


def test_refusals(fh):
    import torch

    def refused(code, call):
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == code, str(e.value)

    for bad in (dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(n_pages=0), dict(n_seqs=0),
                dict(seq_pages=0), dict(n_heads=12), dict(key_heads=4), dict(n_seqs=70000), dict(seq_pages=1 << 26)):
        args = dict(n_pages=4, page_size=16, n_seqs=2, seq_pages=4, n_heads=16, n_kv_heads=8)
        args.update(bad)
        refused(-2, lambda: fh.KvPages(**args))
    import ctypes

    handle = ctypes.c_void_p()
    assert fh.lib().focr_kv_pages_create(fh.default_context().handle, 4, 16, 2, 4, 16, 8, 8, 128, ctypes.byref(handle)) == -3
    kv = fh.KvPages(4, 16, 2, 4)
    refused(-2, lambda: kv.map(2, 0, [0]))
    refused(-2, lambda: kv.map(0, 3, [0, 1]))
    refused(-2, lambda: kv.map(0, -1, [0]))
    refused(-5, lambda: kv.map(0, 0, [4]))
    refused(-5, lambda: kv.map(0, 0, [-2]))
    x = lambda *shape: torch.zeros(shape, device="cuda:0")  # noqa: E731
    lens = int32([0, 0])
    refused(-2, lambda: kv.append(x(3, 8, 64), x(3, 8, 64), lens))  # three rows of two sequences
    refused(-2, lambda: kv.append(x(2, 8, 64), x(3, 8, 64), lens))
    refused(-2, lambda: kv.append(x(3, 8, 64), x(3, 8, 64), int32([0, 0, 0])))  # more sequences than it has
    refused(-2, lambda: kv.append(x(2, 8, 64), x(2, 8, 64), lens.long()))
    refused(-2, lambda: kv.append(x(2, 8, 64), x(2, 8, 64), lens, row_start=int32([0, 2])))
    refused(-2, lambda: kv.qkv_rows(x(2, 32 * 64), x(1, 16, 32, 2), lens))
    refused(-2, lambda: kv.qkv_rows(x(2, 32 * 64), x(2, 16, 32, 2), lens, q=x(1, 16, 64)))
    refused(-2, lambda: kv.attention(x(2, 16, 64), lens, 0))
    refused(-2, lambda: kv.attention(x(2, 16, 64), lens, 65))
    refused(-2, lambda: kv.attention(x(2, 16, 64), lens, 16, sinks=x(8)))
    refused(-2, lambda: kv.attention(x(2, 16, 64), lens, 16, out=x(1, 16, 64)))
    refused(-1, lambda: kv.attention(x(2, 16, 64).cpu(), lens, 16))
    refused(-2, lambda: kv.attention(x(2, 64, 16).transpose(1, 2), lens, 16))
    refused(-2, lambda: kv.dequantize(3, lens))




def test_refusals_of_types(fh):
    # A tensor of fewer bytes than its elements would take would be read past its end.
    import torch

    kv = fh.KvPages(4, 16, 2, 4)
    x = lambda *shape: torch.zeros(shape, device="cuda:0")  # noqa: E731
    lens = int32([0, 0])
    calls = [lambda: kv.attention(x(2, 16, 64).half(), lens, 16),
             lambda: kv.attention(x(2, 16, 64), lens, 16, sinks=x(16).bfloat16()),
             lambda: kv.attention(x(2, 16, 64), lens, 16, out=x(2, 16, 64).half()),
             lambda: kv.append(x(2, 8, 64).half(), x(2, 8, 64), lens),
             lambda: kv.append(x(2, 8, 64), x(2, 8, 64).half(), lens),
             lambda: kv.append(x(2, 8, 64), x(2, 8, 64), lens, row_start=x(3)),
             lambda: kv.qkv_rows(x(2, 32 * 64).half(), x(2, 16, 32, 2), lens),
             lambda: kv.qkv_rows(x(2, 32 * 64), x(2, 16, 32, 2).half(), lens),
             lambda: kv.dequantize(2, lens.float())]
    for call in calls:
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == -2, str(e.value)
    assert kv.refused() == []


def test_page_numbers_are_not_cut_to_32_bits(fh):
    kv = fh.KvPages(4, 16, 2, 4)
    for bad in (np.array([2 ** 32 + 1]), np.array([1.5]), [2 ** 40]):
        with pytest.raises(fh.FocrError) as e:
            kv.map(0, 0, bad)
        assert e.value.code == -5
    kv.map(0, 0, [])
    kv.map(0, 1, np.array([3, -1, 0], dtype=np.int64))
