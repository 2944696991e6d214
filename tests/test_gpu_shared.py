"""Attention of a batch whose sequences begin with the same positions, read once: against 64 bits,
against attention of the same positions sequence by sequence, and what it refuses."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev
from test_gpu_pages import HEADS, attention64, cat, check, decoded, int32, rows_of, starts
from test_gpu_pages_overlap import BATCHES, plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


class Batch:
    """Sequences whose first `shared` positions are one of them's pages, or, with `apart`, those of a
    sequence that is not in the batch (the others have no pages there)."""

    def __init__(self, fh, shared, own, counts, page=64, heads=16, kv_heads=8, key_heads=None, seed=0, scale=1.0, apart=False,
                 ctx=None, prefix=0):
        n, front = len(own), shared // page
        self.shared, self.own, self.counts, self.n, self.heads = shared, own, counts, n, heads
        self.before = [shared + a for a in own]
        self.totals = [b + c for b, c in zip(self.before, counts)]
        back = [-(-(a + c) // page) for a, c in zip(own, counts)]
        n_pages = front + sum(back) + 2
        self.kv = kv = fh.KvPages(n_pages, page, n + apart, front + max(1, max(back)), heads, kv_heads, key_heads=key_heads, ctx=ctx)
        ids = np.random.Generator(np.random.PCG64(seed)).permutation(n_pages)
        at = front
        for i, c in enumerate(back):
            if not apart:
                kv.map(i, 0, ids[:front])
            kv.map(i, front, ids[at:at + c])
            at += c
        self.prefix = n if apart else prefix
        if apart:
            kv.map(n, 0, ids[:front])
        held = [a + c for a, c in zip(own, counts)]
        self.pk, self.pv = gen.normal((shared, kv.key_heads, 64), scale, seed + 1), gen.normal((shared, kv_heads, 64), 1.0, seed + 2)
        self.k, self.v = rows_of(held, kv.key_heads, seed + 3, scale), rows_of(held, kv_heads, seed + 4)
        self.q = rows_of(counts, heads, seed + 5)
        self.sinks = gen.normal((heads,), 1.0, seed + 6)
        if shared:
            kv.append(to_dev(self.pk), to_dev(self.pv), int32([-1] * self.prefix + [0]), row_start=int32([0] * (self.prefix + 1) + [shared]))
        kv.append(cat(self.k), cat(self.v), int32([shared] * n), row_start=starts(held))
        assert kv.refused() == []

    def sequence(self, i):
        """A sequence's keys and values as they are attended to."""
        return (np.concatenate([decoded(self.pk), decoded(self.k[i])]), np.concatenate([decoded(self.pv), decoded(self.v[i])]))

    def shared_call(self, max_len=None, sinks=True, **kw):
        return self.kv.attention_shared(cat(self.q), int32(self.before), max_len or max(self.totals), self.shared, self.prefix,
                                        row_start=starts(self.counts), sinks=to_dev(self.sinks) if sinks else None, **kw)

    def verify(self, got, sinks=True, only=None):
        at = 0
        for i, c in enumerate(self.counts):
            if c and (only is None or i in only):
                k, v = self.sequence(i)
                check(got[at:at + c], *attention64(self.q[i], k, v, self.before[i], self.sinks if sinks else None),
                      f"sequence {i}: {c} rows after {self.before[i]}")
            at += c


@pytest.mark.parametrize("heads,kv_heads,key_heads", HEADS)
@pytest.mark.parametrize("page,shared", [(16, 16), (16, 144), (32, 96), (128, 256)])
def test_a_ragged_batch(fh, heads, kv_heads, key_heads, page, shared):
    # Every row count, own positions from none on, more columns than one tile, one sequence without rows.
    b = Batch(fh, shared, [0, 1, 15, 16, 17, 63, 64, 65, 100, 300], [1, 2, 3, 8, 1, 4, 5, 0, 6, 7], page, heads, kv_heads, key_heads,
              seed=page + heads)
    b.verify(host(b.shared_call()))
    assert b.kv.refused() == []


@pytest.mark.parametrize("sequences,rows", [(1, 1), (1, 3), (1, 8), (2, 1), (3, 1), (4, 1), (5, 1), (8, 1), (9, 1), (16, 1), (17, 1),
                                            (33, 1), (3, 8), (70, 1)])
@pytest.mark.parametrize("key_heads", [8, 16])
def test_batches_of_every_width(fh, sequences, rows, key_heads):
    # From one column of a wave to several tiles of workgroups, without row_start where it can be.
    b = Batch(fh, 320, [(7 * i) % 50 for i in range(sequences)], [rows] * sequences, 64, 16, 8, key_heads, seed=sequences + rows,
              apart=sequences % 2 == 0)
    got = host(b.shared_call(sinks=False))
    b.verify(got, sinks=False)
    if rows == 1:
        again = b.kv.attention_shared(cat(b.q), int32(b.before), max(b.totals), 320, b.prefix)
        assert_bitwise(host(again), got)
    assert b.kv.refused() == []


@pytest.mark.parametrize("shared,page,sequences,rows", [(20480, 128, 3, 2), (6528, 64, 40, 1), (4112, 16, 12, 8)])
def test_long_prefixes(fh, shared, page, sequences, rows):
    b = Batch(fh, shared, [100 + 37 * i % 700 for i in range(sequences)], [rows] * sequences, page, 4, 2, 4, seed=shared)
    b.verify(host(b.shared_call()))


def test_many_rows_over_a_long_prefix(fh):
    # More columns than there are waves for: the prefix is still taken in parts of 4,096 keys.
    n = 140
    b = Batch(fh, 20480, [(7 * i) % 40 for i in range(n)], [8] * n, 128, seed=97)
    b.verify(host(b.shared_call()), only=[0, 77, 139])


@pytest.mark.parametrize("key_heads,own,page", [(8, 40, 16), (16, 40, 64), (16, 1000, 32), (8, 1100, 64)])
def test_many_ragged_sequences(fh, key_heads, own, page):
    # Many sequences, most of one row, some of several, idle, refused or missing a page; own positions
    # from none on, in one part and in several.
    n = 48
    counts = [0 if i % 11 == 5 else 8 if i == 20 else 3 if i % 16 == 7 else 1 for i in range(n)]
    owns = [0 if i == 2 else (own * (7 * i % n) // n if i else own) for i in range(n)]
    b = Batch(fh, 64, owns, counts, page, 16, 8, key_heads, seed=own + key_heads)
    b.before[9] = 63
    at = (64 + owns[30] // 2) // page
    b.kv.map(30, at, [-1])
    got = host(b.shared_call(max_len=64 + own + 8))
    assert b.kv.refused() == [9, 30]
    first = np.concatenate([[0], np.cumsum(counts)])
    assert np.isnan(got[first[9]:first[10]]).all() and np.isnan(got[first[30]:first[31]]).all()
    b.verify(got, only=[i for i in range(n) if i not in (9, 30)])


def test_equals_attention_of_each_sequence(fh):
    # The same positions read by each sequence for itself: within the roundings of both.
    b = Batch(fh, 192, [5, 80, 0], [2, 1, 4], 32, seed=7)
    got, want = host(b.shared_call()), host(b.kv.attention(cat(b.q), int32(b.before), max(b.totals), row_start=starts(b.counts),
                                                           sinks=to_dev(b.sinks)))
    at = 0
    for i, c in enumerate(b.counts):
        _, bound = attention64(b.q[i], *b.sequence(i), b.before[i], b.sinks)
        check(got[at:at + c], want[at:at + c].astype(np.float64), 2 * bound)
        at += c
    assert_bitwise(host(b.shared_call()), got, "another call")
    assert_bitwise(host(b.shared_call(max_len=192 + 96)), got, "a loose bound")
    none = host(b.kv.attention_shared(cat(b.q), int32(b.before), max(b.totals), 0, row_start=starts(b.counts), sinks=to_dev(b.sinks)))
    assert_bitwise(none, want, "nothing is shared")


def test_the_sequences_own_pages_do_not_count_below(fh):
    # A sequence with other pages there than the prefix's sequence, and one with none.
    b = Batch(fh, 64, [3, 20], [1, 2], 32, seed=11)
    got = host(b.shared_call())
    b.kv.map(1, 0, [-1, -1])
    assert_bitwise(host(b.shared_call()), got)
    assert b.kv.refused() == []


def test_peaked_scores_and_far_values(fh):
    b = Batch(fh, 256, [9, 70], [3, 8], seed=13, scale=12.0)
    b.verify(host(b.shared_call()))


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("ratio", [1e6, 1e30])
def test_large_values_without_weight(fh, where, ratio):
    # Large values at scores 100 below the others', in the prefix's or the sequence's part: as
    # FP32 sums are, with no term for them. The bound is that of the accuracy tests (runs of 1,024 at most).
    import test_gpu_pages_accuracy as accuracy

    shared, own, heads = 1088, 60, 2
    n_pages = 20
    kv = fh.KvPages(n_pages, 64, 1, n_pages, heads, heads)
    kv.map(0, 0, list(range(n_pages))[::-1])
    k, v, q = (gen.normal((n, heads, 64), 1.0, 17 + n) for n in (shared + own, shared + own + 1000, 1))
    v = v[:shared + own]
    at = 32 if where == "prefix" else shared + 16
    k[at:at + 16] = accuracy.key_for(q, -100.0)
    v[at:at + 16] *= F32(ratio)
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=int32([0, shared + own]))
    gk, gv = (host(x) for x in kv.dequantize(shared + own, int32([0]), row_start=int32([0, shared + own])))
    got = host(kv.attention_shared(to_dev(q), int32([shared + own - 1]), shared + own, shared))
    want, bound = accuracy.attention64(q, gk, gv, shared + own - 1)
    check(got, want, bound)


@pytest.mark.parametrize("large", [1e4, 3e5])
def test_a_large_query_element_that_meets_no_key(fh, large):
    # Scores come from elements far below the largest one. A query's elements are off by 2^-24 of
    # themselves, and 2^-39 of the largest (by 2^-30 of it among the sequence's own keys), times the key,
    # and scores by the roundings of their own terms' sum and of the exponent.
    shared, own, heads = 1024, 40, 2
    kv = fh.KvPages(18, 64, 1, 18, heads, heads)
    kv.map(0, 0, list(range(18)))
    k, v, q = (gen.normal((n, heads, 64), 1.0, 91 + i) for i, n in enumerate((shared + own, shared + own, 1)))
    k[:, :, 5] = 0
    q[:, :, 5] = large
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=int32([0, shared + own]))
    gk, gv = (host(x).astype(np.float64) for x in kv.dequantize(shared + own, int32([0]), row_start=int32([0, shared + own])))
    got = host(kv.attention_shared(to_dev(q), int32([shared + own - 1]), shared + own, shared)).astype(np.float64)
    eps = 2.0 ** -24
    for h in range(heads):
        s = gk[:, h] @ q[0, h].astype(np.float64) / 8.0
        w = np.exp(s - s.max())
        w /= w.sum()
        step = 2.0 ** -30 * large * np.abs(gk[:, h]).sum(axis=1).max() / 8
        off = step + eps * (16 * (np.abs(gk[:, h]) @ np.abs(q[0, h])).max() / 8 + 8 * np.abs(s).max() + 16)
        bound = w @ np.abs(gv[:, h]) * (2.2 * off + eps * (2 * 1024 + 112))
        over = np.abs(got[0, h] - w @ gv[:, h]) / bound
        assert (over <= 1).all(), f"head {h}: {over.max()} times what is allowed"


@pytest.mark.parametrize("scale", [1e-34, 1e-20, 1e20, 1e35])
def test_values_of_one_small_or_large_magnitude(fh, scale):
    import test_gpu_pages_accuracy as accuracy

    kv = fh.KvPages(6, 64, 1, 6, 2, 2)
    kv.map(0, 0, [4, 2, 0, 1, 3, 5])
    k, v, q = (gen.normal((n, 2, 64), 1.0, 101 + i) for i, n in enumerate((300, 300, 1)))
    v *= F32(scale)
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=int32([0, 300]))
    gk, gv = (host(x) for x in kv.dequantize(300, int32([0]), row_start=int32([0, 300])))
    got = host(kv.attention_shared(to_dev(q), int32([299]), 300, 256))
    check(got, *accuracy.attention64(q, gk, gv, 299))


@pytest.mark.parametrize("gap", [14.0, 20.0, 40.0])
def test_a_first_key_that_takes_the_weight_and_has_no_value(fh, gap):
    # Weights of e^-gap carry the whole result: half the dims' for a value of zeros there.
    import test_gpu_pages_accuracy as accuracy

    for half in (False, True):
        kv = fh.KvPages(18, 64, 1, 18, 2, 2)
        kv.map(0, 0, list(range(18)))
        k, v, q = (gen.normal((n, 2, 64), 1.0, 111 + i) for i, n in enumerate((1100, 1100, 1)))
        k[3] = accuracy.key_for(q, gap)
        v[3] = 0
        if half:
            v[3, :, ::2] = 50.0
        kv.append(to_dev(k), to_dev(v), int32([0]), row_start=int32([0, 1100]))
        gk, gv = (host(x) for x in kv.dequantize(1100, int32([0]), row_start=int32([0, 1100])))
        got = host(kv.attention_shared(to_dev(q), int32([1099]), 1100, 1024))
        check(got, *accuracy.attention64(q, gk, gv, 1099))


def test_non_finite_queries_keys_and_values(fh):
    b = Batch(fh, 64, [4, 9, 30], [2, 1, 3], 16, seed=19)
    flat = np.concatenate(b.q)
    want = host(b.shared_call())
    b.q[0][1, 3, 9] = np.nan
    b.q[2][0, 8, 63] = np.inf
    got = host(b.shared_call())
    nan = np.zeros(flat.shape[:2], bool)
    nan[1, 3] = nan[3, 8] = True
    assert np.array_equal(np.isnan(got).all(axis=2), nan) and np.array_equal(np.isnan(got).any(axis=2), nan)
    assert_bitwise(got[~nan], want[~nan])
    b = Batch(fh, 64, [4, 9], [2, 1], 16, seed=19)
    want = host(b.shared_call())
    bad_k, bad_v = b.pk.copy(), b.pv.copy()
    bad_k[20, 2, 7], bad_v[63, 5, 0] = np.inf, np.nan
    b.kv.append(to_dev(bad_k), to_dev(bad_v), int32([0]), row_start=int32([0, 64]))
    got = host(b.shared_call())
    poisoned = [4, 5, 10, 11]
    assert np.isnan(got[:, poisoned]).all()
    fine = [h for h in range(16) if h not in poisoned]
    assert_bitwise(got[:, fine], want[:, fine])


def test_refused_and_idle_sequences(fh):
    import torch

    # 0 idle, 1 fine, 2 stands before the shared positions, 3 nine rows, 4 longer than max_len, 5 its own page
    # missing, 6 without rows, 7 and 8 fine; a row before the first and one behind the last.
    own, counts = [2, 20, 1, 5, 60, 31, 4, 9, 12], [1, 2, 2, 9, 5, 2, 0, 2, 3]
    b = Batch(fh, 48, own, counts, 16, seed=23, ctx=None)
    kv = b.kv
    kv.map(5, 48 // 16 + 2, [-1])  # its positions 32 .. 47 behind the shared ones
    lens = list(b.before)
    lens[0], lens[2] = -1, 47
    first = 1 + np.concatenate([[0], np.cumsum(counts)])
    rows = int(first[-1]) + 1
    q = gen.normal((rows, 16, 64), 1.0, 29)
    for i, c in enumerate(counts):
        b.q[i] = q[first[i]:first[i] + c]
    out = torch.full((rows, 16, 64), 123.0, device="cuda:0")
    kv.attention_shared(to_dev(q), int32(lens), 48 + 62, 48, 0, row_start=int32(first), sinks=to_dev(b.sinks), out=out)
    assert kv.refused() == [2, 3, 4, 5]
    got = host(out)
    assert (got[[0, 1, rows - 1]] == 123.0).all()  # before the first, the idle one's, behind the last
    for i in (2, 3, 4):
        assert np.isnan(got[first[i]:first[i] + counts[i]]).all(), i
    a = first[5]
    check(got[a:a + 1], *attention64(q[a:a + 1], *b.sequence(5), 48 + 31, b.sinks))  # before its missing page
    assert np.isnan(got[a + 1]).all()
    for i in (1, 7, 8):
        a = first[i]
        check(got[a:a + counts[i]], *attention64(b.q[i], *b.sequence(i), b.before[i], b.sinks), f"sequence {i}")
    # A missing page of the prefix is every sequence's loss; idle ones are not refused for it.
    kv.map(0, 1, [-1])
    got = host(kv.attention_shared(to_dev(q), int32(lens), 48 + 62, 48, 0, row_start=int32(first), sinks=to_dev(b.sinks)))
    assert kv.refused() == [1, 2, 3, 4, 5, 7, 8]
    assert np.isnan(got[first[1]:first[2]]).all() and np.isnan(got[first[8]:first[9]]).all()


@pytest.mark.parametrize("starts_,lens", BATCHES)
@pytest.mark.parametrize("extra", [0, 300])  # sequences without rows before these
def test_overlapping_rows_are_refused_alone(fh, starts_, lens, extra):
    import torch

    n, rows, max_len = 4 + extra, 10, 64
    kv = fh.KvPages(n * 4, 16, n, 4, 16, 8)
    for i in range(extra, n):
        kv.map(i, 0, [4 * i + j for j in range(4)])
    k, v = gen.normal((4 * 40, 8, 64), 1.0, 3), gen.normal((4 * 40, 8, 64), 1.0, 5)
    kv.append(to_dev(k), to_dev(v), int32([0] * n), row_start=int32([0] * extra + [0, 40, 80, 120, 160]))
    assert kv.refused() == []
    if lens[0] == 500:
        lens = [max_len + 1] + lens[1:]
    q = to_dev(gen.normal((rows, 16, 64), 1.0, 7))
    what, nan = plan(starts_, lens, max_len, rows, max_len)
    out = torch.full((rows, 16, 64), 5.0, device="cuda:0")
    kv.attention_shared(q, int32([0] * extra + lens), max_len, 16, extra, row_start=int32([0] * extra + starts_), out=out)
    # The sequences before these have no rows, and so are not refused for standing before position 16.
    assert kv.refused() == [extra + i for i, w in enumerate(what) if w == "refused"]
    got = host(out)
    want = np.full((rows, 16, 64), 5.0, F32)
    want[nan] = np.nan
    for i, w in enumerate(what):
        if isinstance(w, tuple):
            alone = [-1] * n
            alone[extra + i] = lens[i]
            begin, end = w
            one = kv.attention_shared(q, int32(alone), max_len, 16, extra, row_start=int32([begin] * (extra + i + 1) + [end] * (4 - i)))
            want[begin:end] = host(one)[begin:end]
    assert_bitwise(got, want)
    assert kv.refused() == []


def test_groups_in_calls_of_their_own(fh):
    import torch

    # Two prefixes in one batch: a call for each, the other's sequences taking no part, into one output.
    page, shared = 32, [64, 160]
    kv = fh.KvPages(40, page, 6, 8)
    own, counts, group = [3, 40, 0, 17], [1, 2, 1, 3], [0, 1, 1, 0]
    pk, pv = [gen.normal((s, 8, 64), 1.0, 37 + s) for s in shared], [gen.normal((s, 8, 64), 1.0, 41 + s) for s in shared]
    kv.map(4, 0, [0, 1])
    kv.map(5, 0, [2, 3, 4, 5, 6])
    at = 7
    k, v, q = rows_of([a + c for a, c in zip(own, counts)], 8, 43), rows_of([a + c for a, c in zip(own, counts)], 8, 47), rows_of(counts, 16, 53)
    for i in range(4):
        kv.map(i, shared[group[i]] // page, [at, at + 1])
        at += 2
    kv.append(to_dev(np.concatenate(pk)), to_dev(np.concatenate(pv)), int32([-1] * 4 + [0, 0]), row_start=int32([0] * 5 + [64, 224]))
    before = [shared[g] + a for g, a in zip(group, own)]
    kv.append(cat(k), cat(v), int32([shared[g] for g in group]), row_start=starts([a + c for a, c in zip(own, counts)]))
    assert kv.refused() == []
    out = torch.zeros(sum(counts), 16, 64, device="cuda:0")
    for g in range(2):
        lens = [b if x == g else -1 for b, x in zip(before, group)]
        kv.attention_shared(cat(q), int32(lens), 224, shared[g], 4 + g, row_start=starts(counts), out=out)
    got, at = host(out), 0
    for i, c in enumerate(counts):
        kk, vv = np.concatenate([decoded(pk[group[i]]), decoded(k[i])]), np.concatenate([decoded(pv[group[i]]), decoded(v[i])])
        check(got[at:at + c], *attention64(q[i], kk, vv, before[i], None), f"sequence {i}")
        at += c
    assert kv.refused() == []


def test_offsets_past_32_bits(fh):
    # 2.4 GB of key codes: the prefix's last page, and a sequence's own, do not fit 32 bits.
    page, n_pages = 4096, 580
    kv = fh.KvPages(n_pages, page, 2, 2, 16, 8, key_heads=16)
    kv.map(0, 0, [n_pages - 1, 0])
    kv.map(1, 1, [n_pages - 2])
    pk, pv = gen.normal((page, 16, 64), 1.0, 59), gen.normal((page, 8, 64), 1.0, 61)
    k, v, q = rows_of([5, 50], 16, 67), rows_of([5, 50], 8, 71), rows_of([2, 1], 16, 73)
    kv.append(to_dev(pk), to_dev(pv), int32([0]), row_start=int32([0, page]))
    kv.append(cat(k), cat(v), int32([page, page]), row_start=starts([5, 50]))
    got = host(kv.attention_shared(cat(q), int32([page + 3, page + 49]), page + 50, page, row_start=starts([2, 1])))
    for i, (lo, hi) in enumerate(((0, 2), (2, 3))):
        kk, vv = np.concatenate([decoded(pk), decoded(k[i])]), np.concatenate([decoded(pv), decoded(v[i])])
        check(got[lo:hi], *attention64(q[i], kk, vv, [page + 3, page + 49][i], None), f"sequence {i}")
    assert kv.refused() == []


def test_captured_steps(fh):
    # Lengths are advanced by the graph; the eager calls between its replays use another context.
    import torch

    ctx = fh.Context(0)
    steps, n = 20, 5
    b = Batch(fh, 128, [0, 3, 15, 40, 7], [steps] * n, 16, seed=79, ctx=ctx)
    other = Batch(fh, 128, [0, 3, 15, 40, 7], [steps] * n, 16, seed=79)
    lens, q, out = int32(b.before), torch.zeros(n, 16, 64, device="cuda:0"), torch.zeros(n, 16, 64, device="cuda:0")
    sinks, most = to_dev(b.sinks), max(b.totals)
    b.kv.attention_shared(q, lens, most, 128, sinks=sinks)  # the scratch grows uncaptured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        b.kv.attention_shared(q, lens, most, 128, sinks=sinks, out=out)
        lens.add_(1)
    ctx.use_stream(torch.cuda.current_stream())
    for step in range(steps):
        x = to_dev(gen.normal((n, 16, 64), 1.0, 83 + step))
        q.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = other.kv.attention_shared(x, int32([t + step for t in b.before]), most, 128, sinks=sinks)
        assert_bitwise(host(out), host(want), f"step {step}")
    assert b.kv.refused() == []


def test_two_streams_and_contexts(fh):
    import torch

    sets = []
    for i in range(2):
        ctx, stream = fh.Context(0), torch.cuda.Stream()
        b = Batch(fh, 512, [10 * i + 3 * j for j in range(20)], [1] * 20, 64, seed=89 + i, ctx=ctx)
        sets.append((ctx, stream, b, cat(b.q), int32(b.before), starts(b.counts), to_dev(b.sinks)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (ctx, stream, b, q, lens, start, sinks) in enumerate(sets):
            with torch.cuda.stream(stream):
                ctx.use_stream(stream)
                got[i].append(b.kv.attention_shared(q, lens, max(b.totals), 512, row_start=start, sinks=sinks))
    torch.cuda.synchronize()
    for g, s in zip(got, sets):
        for t in g:
            assert_bitwise(host(t), host(g[0]))
        s[2].verify(host(g[0]))


def test_refusals(fh):
    import torch

    def refused(code, call):
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == code, str(e.value)

    kv = fh.KvPages(8, 32, 2, 4)
    q, lens = torch.zeros(2, 16, 64, device="cuda:0"), int32([64, 64])
    refused(-2, lambda: kv.attention_shared(q, lens, 128, 48))  # not whole pages
    refused(-2, lambda: kv.attention_shared(q, lens, 128, 160))  # more than a sequence's pages
    refused(-2, lambda: kv.attention_shared(q, lens, 128, -32))
    refused(-2, lambda: kv.attention_shared(q, lens, 64, 64))  # max_len leaves no own position
    refused(-2, lambda: kv.attention_shared(q, lens, 129, 64))
    refused(-2, lambda: kv.attention_shared(q, lens, 128, 64, prefix=2))
    refused(-2, lambda: kv.attention_shared(q, lens, 128, 64, prefix=-1))
    refused(-2, lambda: kv.attention_shared(q, int32([64]), 128, 64))
    refused(-2, lambda: kv.attention_shared(q.half(), lens, 128, 64))
    refused(-2, lambda: kv.attention_shared(q, lens, 128, 64, out=q[:1]))
    empty = kv.attention_shared(q[:0], int32([]), 128, 64)
    assert empty.shape == (0, 16, 64)
