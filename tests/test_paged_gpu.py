"""The paged key/value cache: block tables and slot maps, release, append and attention, against plain NumPy in 64 bits.

Attention's tolerance, per element, with A = sum_j p_j |v_j|: the output's rounding u |o| (u = half the type's step), the
weights' rounding where a product takes them in half precision (u A, and 2^-25 |v| for weights below fp16's normal range), the
scores' error d (fp32 dot products of D terms) in the weights and in their sum, and (n + 8) 2^-24 of both fp32 sums over n keys
with the exponential's error."""
import ctypes

import numpy as np
import pytest

from tests.test_ops_gpu import DTYPES, dev, no_device_flag, rnd

pytestmark = pytest.mark.gpu
U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def mt():
    import mytorch_b200 as m
    return m


def device_flag(mt):
    f = ctypes.c_int(0)
    mt._lib.device_flag_read(ctypes.byref(f), mt.stream())
    return f.value


def i32(mt, a):
    return mt.DeviceArray.from_numpy(np.asarray(a, np.int32), "int32")


# ------------------------------------------------------------------ tables ----
def tables_by_hand(held, fresh, tables, free, page, rows):
    """One request and one page after the other."""
    tables, free, width = tables.copy(), list(free), tables.shape[1]
    starts, position, slot, short = [0], np.zeros(rows, np.int32), np.full(rows, -1, np.int32), False
    for r, (h, f) in enumerate(zip(np.maximum(held, 0), np.maximum(fresh, 0))):
        first, last = -(-h // page), -(-(h + f) // page)
        for at in range(first, min(last, width)):
            tables[r, at] = free.pop() if free else -1
        short |= (tables[r, first:last] < 0).any() or last > width
        for i in range(f):
            if starts[-1] + i < rows:
                at = (h + i) // page
                position[starts[-1] + i] = h + i
                if at < width and tables[r, at] >= 0:
                    slot[starts[-1] + i] = tables[r, at] * page + (h + i) % page
        starts.append(starts[-1] + f)
    return tables, np.array(starts), np.maximum(held, 0) + np.maximum(fresh, 0), position, slot, len(free), short


def check_tables(mt, held, fresh, page, width, spare, rows, short=False):
    held, fresh = np.asarray(held), np.asarray(fresh)
    r = np.random.default_rng(len(held))
    own = [min(-(-max(h, 0) // page), width) for h in held]
    pool = r.permutation(sum(own) + spare)
    tables, at = np.full((len(held), width), -1, np.int32), 0
    for row, n in zip(tables, own):
        row[:n] = pool[at:at + n]
        at += n
    free = np.concatenate([pool[at:], np.full(at, -7)])
    want = tables_by_hand(held, fresh, tables, pool[at:], page, rows)
    assert want[-1] == short
    T, args = i32(mt, tables), [i32(mt, held), i32(mt, fresh)]
    out = None
    for again in range(2):                       # the same call twice is the same step
        out = mt.fused_ops.fused_paged_tables(*args, T, i32(mt, free), i32(mt, [len(pool) - at]), page, rows=rows, out=out)
        for name, got, w in zip(("starts", "kv_len", "position", "slot", "left"), out, want[1:]):
            assert np.array_equal(got.numpy().reshape(-1), np.asarray(w).reshape(-1)), name
        assert np.array_equal(T.numpy(), want[0])
    assert device_flag(mt) == (3 if short else 0)


@pytest.mark.parametrize("page", [1, 7, 16, 256])
@pytest.mark.parametrize("requests", [1, 5, 1023, 1025, 3000])
def test_tables(mt, requests, page):
    r = np.random.default_rng(page * requests)
    held, fresh = r.integers(0, 60, requests), r.integers(0, 4, requests)
    held[0], fresh[-1] = 0, 40                   # an empty request, one that takes several pages
    fresh[requests // 2] = 0
    width = -(-101 // page)
    need = int((-(-(held + fresh) // page) - -(-held // page)).sum())
    check_tables(mt, held, fresh, page, width, need + 2, int(fresh.sum()) + 3)
    check_tables(mt, held, fresh, page, width, need, max(1, int(fresh.sum())))          # the last page, no padding


def test_tables_of_one_long_request(mt):
    check_tables(mt, [0], [5000], 16, 400, 400, 5000)
    check_tables(mt, [4095, 0, 17], [1, 0, 2000], 64, 70, 40, 2001)


def test_tables_without_enough_pages(mt):
    check_tables(mt, [3, 16, 30], [20, 1, 10], 16, 8, 2, 40, short=True)                # the third request gets none
    check_tables(mt, [3, 16, 30], [20, 1, 10], 16, 2, 9, 40, short=True)                # the table is too narrow for it
    check_tables(mt, [3, -4, 30], [20, -1, 2], 16, 8, 5, 30)                            # negative counts are zero


def test_tables_at_most_requests(mt):
    check_tables(mt, np.full(8192, 15), np.full(8192, 2), 16, 2, 8192, 16384)


def test_tables_more_tokens_than_rows(mt):
    F = mt.fused_ops
    out = F.fused_paged_tables(i32(mt, [0]), i32(mt, [9]), i32(mt, [[-1]]), i32(mt, [4]), i32(mt, [1]), 16, rows=5)
    assert list(out[3].numpy()) == [64, 65, 66, 67, 68] and device_flag(mt) == 3


@pytest.mark.parametrize("requests,width,page", [(1, 1, 16), (7, 5, 3), (2000, 6, 8), (8192, 2, 16)])
def test_release(mt, requests, width, page):
    r = np.random.default_rng(requests)
    kv = r.integers(0, width * page + 1, requests)
    done = r.random(requests) < 0.4
    done[0] = True
    n = -(-kv // page)
    pool = r.permutation(int(n.sum()) + 4)
    tables, at = np.full((requests, width), -1, np.int32), 0
    for row, m in zip(tables, n):
        row[:m] = pool[at:at + m]
        at += m
    if n[0] > 1:
        tables[0, 0] = -1                                        # a page that was never there does not come back
    free = np.concatenate([pool[at:], np.full(at, -7)]).astype(np.int32)
    gone = [p for row, d in zip(tables, done) if d for p in row if p >= 0]
    T, KV, L, NF = i32(mt, tables), i32(mt, kv), i32(mt, free), i32(mt, [4])
    mt.fused_ops.fused_paged_release(i32(mt, done), T, KV, L, NF, page)
    assert NF.item() == 4 + len(gone) and list(L.numpy()[:NF.item()]) == list(free[:4]) + gone
    assert np.array_equal(T.numpy(), np.where(done[:, None], -1, tables)) and np.array_equal(KV.numpy(), np.where(done, 0, kv))
    no_device_flag(mt)


# ------------------------------------------------------------------ append ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,D,page,pages", [(1, 1, 64, 16, 2), (33, 3, 128, 7, 9), (500, 12, 64, 64, 9), (5, 2, 10, 3, 4), (3, 1, 1, 1, 5)])
def test_append(mt, dtype, rows, heads, D, page, pages):
    r = np.random.default_rng(rows)
    new, pools = (rnd(r.standard_normal((2, rows, heads, D)), dtype), rnd(r.standard_normal((2, pages, heads, page, D)), dtype))
    slot = r.permutation(pages * page)[:rows].astype(np.int32)
    slot = np.concatenate([slot, np.full(rows - len(slot), -1, np.int32)])
    slot[rows // 2] = -1
    K, V = (dev(mt, a, dtype) for a in pools)
    mt.fused_ops.fused_paged_append(dev(mt, new[0], dtype), dev(mt, new[1], dtype), K, V, i32(mt, slot))
    want = pools.copy()
    for i, s in enumerate(slot):
        if s >= 0:
            want[:, s // page, :, s % page] = new[:, i]
    assert np.array_equal(K.numpy(), want[0]) and np.array_equal(V.numpy(), want[1])
    no_device_flag(mt)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_reads_a_projection_in_place(mt, dtype):
    """Keys and values as column slices of a wider row, at an odd offset of the row too; a slot beyond the pool is left out."""
    r = np.random.default_rng(2)
    St = mt._lib.Strides3
    for lead in (0, 1):
        wide = rnd(r.standard_normal((6, 3 * 2 * 64 + lead)), dtype)
        W, item = dev(mt, wide, dtype), 4 if dtype == "float32" else 2
        K, V = (dev(mt, np.zeros((4, 2, 5, 64)), dtype) for _ in range(2))
        view = lambda at: mt.DeviceArray(W.ptr + (lead + at) * item, (6, 2, 64), dtype, base=W)
        st = St(0, 3 * 64, wide.shape[1])
        slot = np.array([3, 19, 20, 0, -1, 7])
        mt.fused_ops.fused_paged_append(view(64), view(128), K, V, i32(mt, slot), strides=(st, st))
        assert device_flag(mt) == 3
        want = np.zeros((2, 4, 2, 5, 64), np.float32)
        for i, s in enumerate(slot):
            if 0 <= s < 20:
                want[:, s // 5, :, s % 5] = wide[i, lead:].reshape(2, 3, 64)[:, 1:].swapaxes(0, 1)
        assert np.array_equal(K.numpy(), want[0]) and np.array_equal(V.numpy(), want[1])


# --------------------------------------------------------------- attention ----
class Step:
    """A batch on the host: requests as (keys, new rows) in pages of a shuffled pool whose unused rows are NaN."""

    def __init__(self, requests, heads, kv_heads, D, page, dtype, seed=0, pad=3, scale=1.0):
        r = np.random.default_rng(seed)
        self.requests, self.heads, self.kv_heads, self.D, self.page, self.dtype = requests, heads, kv_heads, D, page, dtype
        n = [-(-kv // page) for kv, _ in requests]
        self.pages, self.width = sum(n) + 2, max(n) + 1
        self.tables = np.full((len(requests), self.width), -1, np.int32)
        self.k = np.full((self.pages, kv_heads, page, D), np.nan, np.float32)
        self.v = self.k.copy()
        order, at = r.permutation(self.pages), 0
        for row, m, (kv, _) in zip(self.tables, n, requests):
            row[:m] = order[at:at + m]
            at += m
            j = np.arange(kv)
            self.k[row[j // page], :, j % page] = rnd(r.standard_normal((kv, kv_heads, D)) * scale, dtype)
            self.v[row[j // page], :, j % page] = rnd(r.standard_normal((kv, kv_heads, D)), dtype)
        self.starts = np.concatenate([[0], np.cumsum([m for _, m in requests])]).astype(np.int32)
        self.rows = int(self.starts[-1]) + pad
        self.q = rnd(r.standard_normal((self.rows, heads, D)) * scale, dtype)

    def gather(self, r, h):
        j = np.arange(self.requests[r][0])
        p = self.tables[r, j // self.page]
        ok = (p >= 0) & (p < self.pages)
        at = (np.where(ok, p, 0), h // (self.heads // self.kv_heads), j % self.page)
        return self.k[at].astype(np.float64), self.v[at].astype(np.float64), ok

    def want(self, scale=None):
        """(o, allowed error) of the rows that requests have."""
        scale = self.D ** -0.5 if scale is None else scale
        u, half = U[self.dtype], self.dtype != "float32"
        out = np.zeros((self.starts[-1], self.heads, self.D))
        tol = np.zeros_like(out)
        for r, (kv, m) in enumerate(self.requests):
            for h in range(self.heads):
                k, v, ok = self.gather(r, h)
                q = self.q[self.starts[r]:self.starts[r + 1], h].astype(np.float64)
                seen = ok & (np.arange(kv) <= np.arange(kv - m, kv)[:, None])
                with np.errstate(invalid="ignore"):
                    s = np.where(seen, q @ k.T * scale, -np.inf)
                    d = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0).max(-1, initial=0, keepdims=True) * (self.D + 4) * 2.0 ** -24
                top = s.max(-1, initial=-np.inf, keepdims=True)
                p = np.exp(s - np.where(np.isfinite(top), top, 0))
                l = p.sum(-1, keepdims=True)
                p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
                vv = np.where(seen.any(0)[:, None], v, 0)
                rows = slice(self.starts[r], self.starts[r + 1])
                out[rows, h] = p @ vv
                A = p @ np.abs(vv)
                n = seen.sum(-1, keepdims=True)
                tol[rows, h] = (u * np.abs(out[rows, h]) + ((u if half else 0) + 2 * d + 2 * (n + 8) * 2.0 ** -24) * A
                                + (2.0 ** -25 * (seen @ np.abs(vv)) + 2.0 ** -25 if self.dtype == "float16" else 0) + 1e-30)
        return out, tol

    def run(self, mt, max_new=None, scale=None, q=None, strides=None):
        fill = np.full(self.q.shape, 7.0, np.float32)
        self.O = dev(mt, fill, self.dtype)
        q = dev(mt, self.q, self.dtype) if q is None else q
        mt.fused_ops.fused_paged_attention(q, dev(mt, self.k, self.dtype), dev(mt, self.v, self.dtype), i32(mt, self.tables),
                                           i32(mt, self.starts), i32(mt, [kv for kv, _ in self.requests]), max_new=max_new,
                                           softmax_scale=scale, out=self.O, strides=strides)
        got = self.O.numpy().astype(np.float64)
        assert (got[self.starts[-1]:] == 7).all(), "rows that no request has"
        return got[:self.starts[-1]]

    def check(self, mt, **how):
        got = self.run(mt, **how)
        want, tol = self.want(how.get("scale"))
        assert np.isfinite(got).all()
        over = np.abs(got - want) / tol
        assert over.max(initial=0) <= 1, f"{over.max():.2f} times the tolerance at {np.unravel_index(over.argmax(), over.shape)}"
        return got


ONE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (127, 1), (129, 1), (300, 1)]
FEW = [(4, 4), (1, 1), (70, 3), (0, 0), (33, 2), (130, 4), (9, 0), (257, 4)]
MIXED = [(200, 1), (150, 150), (5, 5), (400, 90), (64, 1), (0, 0), (129, 128), (1, 1), (260, 33)]
SHAPES = [(1, 1, 64), (4, 4, 128), (5, 1, 128), (10, 2, 64), (14, 2, 128), (3, 1, 64), (40, 1, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("batch,max_new", [(ONE, 1), (FEW, 4), (MIXED, 150)])
def test_attention(mt, dtype, heads, kv_heads, D, batch, max_new):
    Step(batch, heads, kv_heads, D, 16, dtype).check(mt, max_new=max_new)
    no_device_flag(mt)


# Pages smaller than a load, odd, as large as a tile and larger; one that ends inside every tile.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 3, 24, 100, 128, 256])
@pytest.mark.parametrize("batch,max_new", [(ONE, 1), (MIXED, 150)])
def test_attention_page_sizes(mt, dtype, page, batch, max_new):
    Step(batch, 4, 2, 64, page, dtype, seed=page).check(mt, max_new=max_new)
    Step(batch[3:], 2, 2, 128, page, dtype, seed=page + 1).check(mt, max_new=max_new)
    no_device_flag(mt)


# One request alone and few of them: the keys are split over the GPU and joined.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,max_new", [([(9000, 1)], 1), ([(5000, 2), (1, 1), (3000, 2)], 2), ([(6000, 70)], 70), ([(3000, 300), (2500, 1)], 300)])
@pytest.mark.parametrize("heads,kv_heads,D", [(1, 1, 128), (5, 1, 64)])
def test_attention_long(mt, dtype, batch, max_new, heads, kv_heads, D):
    Step(batch, heads, kv_heads, D, 32, dtype, seed=1).check(mt, max_new=max_new)
    no_device_flag(mt)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many_requests(mt, dtype):
    """More requests than a block has threads, most of them tiny; every row is the same whatever stands beside it."""
    r = np.random.default_rng(3)
    batch = [(int(n), min(int(n), int(f))) for n, f in zip(r.integers(0, 40, 1500), r.integers(0, 3, 1500))]
    Step(batch, 2, 1, 64, 8, dtype).check(mt, max_new=2)
    Step(batch[:700] + [(90, 80)] + batch[700:], 2, 1, 64, 8, dtype).check(mt, max_new=80)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [None, 1, 3, 1000])
def test_max_new_is_a_hint_only(mt, dtype, max_new):
    Step(MIXED, 4, 2, 64, 16, dtype).check(mt, max_new=max_new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 40])
def test_fewer_keys_than_new_rows(mt, dtype, max_new):
    """The first rows of such a request see no key and are 0."""
    step = Step([(3, 7), (0, 4), (20, 5), (0, 2), (70, 90)], 4, 2, 64, 16, dtype)
    got = step.check(mt, max_new=max_new)
    assert (got[:4] == 0).all() and (got[7:11] == 0).all() and (got[18:38] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 40])
def test_scale_and_large_scores(mt, dtype, max_new):
    """Scores up to some hundreds: the maximum moves by far more than a rescale's threshold between tiles."""
    Step([(700, 1), (300, 20)], 4, 2, 128, 16, dtype, scale=4.0).check(mt, max_new=max_new)
    Step([(700, 1), (300, 20)], 4, 2, 128, 16, dtype, scale=0.3).check(mt, max_new=max_new, scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 40])
@pytest.mark.parametrize("lead", [0, 1])
def test_queries_in_a_projection(mt, dtype, max_new, lead):
    step = Step([(90, 4), (40, 30)], 4, 4, 64, 16, dtype)
    wide = np.zeros((step.rows, 4, 3 * 64), np.float32)
    wide[:, :, :64] = step.q
    flat = np.concatenate([np.zeros(lead, np.float32), wide.reshape(-1)])
    W = dev(mt, flat, dtype)
    view = mt.DeviceArray(W.ptr + lead * W.itemsize, step.q.shape, dtype, base=W)
    step.check(mt, max_new=max_new, q=view, strides=mt._lib.Strides3(0, 3 * 64, 4 * 3 * 64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 60])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_reach_only_those_that_see_them(mt, dtype, max_new, bad):
    """A key or value that is not finite makes the rows that see it not finite, and no other one."""
    batch = [(200, 60), (150, 1), (90, 3)]
    for which in ("k", "v"):
        step = Step(batch, 4, 2, 64, 16, dtype)
        clean, tol = step.want()
        at = 170                                               # seen by the first request's new rows from 30 on
        pool = getattr(step, which)
        pool[step.tables[0, at // 16], 1, at % 16, 5] = bad
        got = step.run(mt, max_new=max_new)
        hit = np.zeros(got.shape[:2], bool)
        hit[30:60, 2:] = True
        assert (np.abs(got - clean) <= tol)[~hit].all()
        if which == "v":
            assert (~np.isfinite(got[hit][:, 5])).all() and np.isfinite(np.delete(got[hit], 5, 1)).all()
        elif np.isnan(bad):
            assert np.isnan(got[hit]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 40])
def test_keys_that_count_for_nothing(mt, dtype, max_new):
    """Scores of the type's lowest value and of -inf."""
    batch = [(100, 1), (80, 20), (40, 1)]
    step = Step(batch, 2, 1, 64, 16, dtype)
    step.q[:, :, 0] = 1
    j = np.arange(0, 30)
    step.k[step.tables[0, j // 16], 0, j % 16, 0] = -np.inf
    step.k[step.tables[1, j // 16], 0, j % 16, 0] = -(3e38 if dtype != "float16" else 65504)
    j = np.arange(40)
    step.k[step.tables[2, j // 16], 0, j % 16, 0] = -np.inf     # nothing is left of the third request
    with np.errstate(invalid="ignore"):
        want, _ = step.want()
    got = step.run(mt, max_new=max_new)
    assert np.isfinite(got).all() and (got[21] == 0).all()
    # values below 4: output and weights round by 4 u each; the keys that count have sums |q||k| / 8 below 12, so scores are off by
    # less than 12 * 68 * 2^-24, and 100 keys' sums by 108 * 2^-24, both twice in a mean of values below 1
    assert (np.abs(got - want) <= 8 * U[dtype] + 2 * (12 * 68 + 108) * 2.0 ** -24)[:21].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 60])
def test_pages_outside_the_pool_are_left_out(mt, dtype, max_new):
    step = Step([(200, 60), (150, 1), (90, 3)], 4, 2, 64, 16, dtype)
    step.tables[0, 3], step.tables[1, 0], step.tables[2, 1] = -1, step.pages, 2 ** 31 - 1
    step.check(mt, max_new=max_new)
    assert device_flag(mt) == 3


@pytest.mark.parametrize("max_new", [1, 60])
def test_lengths_beyond_the_table(mt, max_new):
    """What lies behind the table's last entry is not there."""
    step = Step([(90, 3)], 2, 1, 64, 16, "float16")
    step.tables = step.tables[:, :4]
    step.width = 4
    O = dev(mt, np.zeros(step.q.shape), "float16")
    mt.fused_ops.fused_paged_attention(dev(mt, step.q, "float16"), dev(mt, step.k, "float16"), dev(mt, step.v, "float16"),
                                       i32(mt, step.tables), i32(mt, step.starts), i32(mt, [90]), max_new=max_new, out=O)
    step.requests = [(64, 3)]
    k, v, _ = step.gather(0, 0)
    s = np.einsum("mhd,nd->mhn", step.q[:3].astype(np.float64), k) / 8
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("mhn,nd->mhd", p / p.sum(-1, keepdims=True), v)
    assert np.abs(O.numpy()[:3] - want).max() <= 2 * U["float16"] * 4 and device_flag(mt) == 3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 60])
def test_twice_the_same_bits(mt, dtype, max_new):
    step = Step([(3000, 60), (150, 1), (2090, 3)], 5, 1, 128, 16, dtype)
    assert np.array_equal(step.run(mt, max_new=max_new), step.run(mt, max_new=max_new))


def test_no_requests_and_no_rows(mt):
    z = lambda *s: mt.DeviceArray.zeros(s, "float16")
    pools = z(2, 1, 16, 64), z(2, 1, 16, 64)
    out = mt.fused_ops.fused_paged_attention(z(3, 1, 64), *pools, i32(mt, np.zeros((1, 1))), i32(mt, [0, 0]), i32(mt, [0]))
    assert (out.numpy() == 0).all()
    mt.fused_ops.fused_paged_attention(z(0, 1, 64), *pools, i32(mt, np.zeros((1, 1))), i32(mt, [0, 0]), i32(mt, [0]))
    mt.fused_ops.fused_paged_append(z(0, 1, 64), z(0, 1, 64), *pools, i32(mt, np.zeros(0)))
    no_device_flag(mt)


# Rows that lie apart from each other, at odd addresses too, and pools with the heads inside a page's rows.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 150])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (5, 1, 128), (2, 2, 128)])
@pytest.mark.parametrize("lead,gap", [(0, 64), (8, 8), (1, 3)])
@pytest.mark.parametrize("rows_first", [False, True])
def test_strides(mt, dtype, max_new, heads, kv_heads, D, lead, gap, rows_first):
    from mytorch_b200 import _lib
    from mytorch_b200.array import stream
    step = Step(MIXED, heads, kv_heads, D, 16, dtype, seed=lead)
    wide = np.full((step.rows, heads * D + gap), 7.0, np.float32)
    wide[:, :heads * D] = step.q.reshape(step.rows, -1)
    flat = np.concatenate([np.full(lead, 7.0, np.float32), wide.reshape(-1)])
    Q, O = dev(mt, flat, dtype), dev(mt, np.full(flat.shape, 7.0), dtype)
    at, st = lead * Q.itemsize, _lib.Strides3(0, D, heads * D + gap)
    pools = [p.swapaxes(1, 2) if rows_first else p for p in (step.k, step.v)]
    K, V = (dev(mt, np.ascontiguousarray(p), dtype) for p in pools)
    sp = _lib.Strides3(kv_heads * 16 * D, D, kv_heads * D) if rows_first else _lib.Strides3(kv_heads * 16 * D, 16 * D, D)
    ints = [i32(mt, a) for a in (step.tables, step.starts, [kv for kv, _ in step.requests])]       # kept until the call is queued
    _lib.attn_paged(Q.ptr + at, K.ptr, V.ptr, O.ptr + at, st, sp, st, *[a.ptr for a in ints], len(step.requests), step.width, step.rows, max_new, heads, kv_heads, D, 16,
                    step.pages, D ** -0.5, Q.code, stream())
    flat = O.numpy().astype(np.float64)
    got = flat[lead:].reshape(step.rows, -1)
    assert (flat[:lead] == 7).all() and (got[:, heads * D:] == 7).all() and (got[step.starts[-1]:] == 7).all()
    want, tol = step.want()
    assert (np.abs(got[:step.starts[-1], :heads * D].reshape(want.shape) - want) <= tol).all()
    no_device_flag(mt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [1, 50])
def test_rows_before_the_first_request(mt, dtype, max_new):
    """starts need not begin at row 0, and a request may end where the rows do."""
    step = Step([(70, 50), (33, 1), (9, 9)], 4, 2, 64, 16, dtype, pad=0)
    want, tol = step.want()
    n = step.rows
    q = np.concatenate([np.full((5, 4, 64), np.nan, np.float32), step.q])
    O = dev(mt, np.full(q.shape, 7.0), dtype)
    mt.fused_ops.fused_paged_attention(dev(mt, q, dtype), dev(mt, step.k, dtype), dev(mt, step.v, dtype), i32(mt, step.tables),
                                       i32(mt, step.starts + 5), i32(mt, [kv for kv, _ in step.requests]), max_new=max_new, out=O)
    got = O.numpy()
    assert (got[:5] == 7).all() and (np.abs(got[5:] - want) <= tol).all() and len(got) == n + 5
    no_device_flag(mt)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_offsets_beyond_32_bits(mt, dtype):
    """A pool of 70000 pages (9 or 18 GB with its values): its last pages lie more than 2^31 elements from its start."""
    F, pages, Hk, page, D = mt.fused_ops, 70000, 4, 64, 128
    big = [mt.DeviceArray.empty((pages, Hk, page, D), dtype) for _ in range(2)]
    small = [mt.DeviceArray.zeros((8, Hk, page, D), dtype) for _ in range(2)]
    r = np.random.default_rng(0)
    lens, fresh = [150, 200], [1, 60]
    n = sum(lens)
    tables = np.array([[3, 1, 6, -1], [0, 7, 2, 5]], np.int32)
    pos = np.concatenate([np.arange(k) for k in lens])
    row = np.repeat([0, 1], lens)
    slot = tables[row, pos // page] * page + pos % page
    k, v = (dev(mt, r.standard_normal((n, Hk, D)), dtype) for _ in range(2))
    q = dev(mt, r.standard_normal((sum(fresh), 8, D)), dtype)
    F.fused_paged_append(k, v, *small, i32(mt, slot))
    F.fused_paged_append(k, v, *big, i32(mt, slot + (pages - 8) * page))
    for max_new in (1, 60):
        ask = lambda pools, t: F.fused_paged_attention(q, *pools, i32(mt, t), i32(mt, [0, 1, 61]), i32(mt, lens), max_new=max_new).numpy()
        assert np.array_equal(ask(big, np.where(tables >= 0, tables + pages - 8, -1)), ask(small, tables))
    no_device_flag(mt)


def bits(mt):
    """Outputs of every kernel, on whatever stream and with whatever overlap is set."""
    return [Step(batch, 4, 2, D, 16, dtype).run(mt, max_new=m) for dtype in DTYPES for D in (64, 128)
            for batch, m in (([(3000, 1), (150, 1)], 1), (MIXED, 150), ([(40, 1), (9, 1)], 1))]


def test_without_overlap_and_on_another_stream(mt, tmp_path):
    """Kernels that start before their predecessor has ended read nothing that it writes: the same bits with the overlap
    off (MT_PDL=0, read once per process), and on a stream of the caller's."""
    import os
    import subprocess
    import sys
    from mytorch_b200 import _lib, array
    want = bits(mt)
    code = f"import mytorch_b200 as mt, numpy as np, tests.test_paged_gpu as t; np.savez({str(tmp_path / 'x.npz')!r}, *t.bits(mt))"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    child = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, MT_PDL="0"), capture_output=True, text=True, timeout=300)
    assert child.returncode == 0, child.stderr[-2000:]
    with np.load(tmp_path / "x.npz") as z:
        assert all(np.array_equal(z[f"arr_{i}"], w) for i, w in enumerate(want))
    mine, before = ctypes.c_void_p(), array.stream()
    array.synchronize()
    _lib.stream_create(ctypes.byref(mine))
    array.set_stream(mine)
    try:
        assert all(np.array_equal(a, b) for a, b in zip(bits(mt), want))
        array.synchronize()
    finally:
        array.set_stream(before)
    _lib.stream_destroy(mine)
