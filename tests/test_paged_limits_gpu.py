"""The paged cache's entry points at the limits of what they take."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def mt():
    import mytorch_b200 as m
    return m


def child(code):
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    return run.stdout


# The kernel's shared memory is 8 bytes a request and 512 besides: 48 KB, where a launch has to ask for more, lies at 6080
# requests. Each first in a process of its own, as one call that asked helps all later ones.
@pytest.mark.parametrize("requests", [6080, 6081, 6144, 6145, 8192])
def test_tables_as_a_process_first_call(requests):
    child("import numpy as np, mytorch_b200 as mt, tests.test_paged_gpu as t;"
          f"t.check_tables(mt, np.full({requests}, 15), np.full({requests}, 2), 16, 2, {requests}, {2 * requests})")


@pytest.mark.parametrize("dtype,max_new", [("float16", 1), ("float16", 40), ("bfloat16", 40), ("float32", 1)])
def test_the_longest_request_that_a_table_can_hold(mt, dtype, max_new):
    """2^31 - 21 keys, the last ones in a tile that ends where 32-bit numbers do. Entries of the table may be equal: four pages over
    and over, and a last one whose scores are 22 higher, so that its 11 keys weigh more than all others together.

    Tolerance: an accumulator takes k sums one after the other over a block's share of the keys, each off by at most 2^-23 of it (the
    tensor cores cut off, others round): tiles of 128 keys, a share of 2^24 / 444 of them with 4 sums each (few rows, half),
    2^24 / 148 with 8 (many rows); 2^26 / 592 tiles of 32 keys with 8 (fp32). The weights' sum has no more, and 4 u covers the
    roundings of weights and output. Scores are off by less than 2 (|q| |k| D 2^-24): 80 * 64 * 2^-24, far below."""
    from tests.test_ops_gpu import dev, no_device_flag, rnd
    from tests.test_paged_gpu import U, i32
    D, page = 64, 16
    width = 2 ** 27 - 1
    keys = width * page - 5
    r = np.random.default_rng(0)
    k, v = (rnd(r.standard_normal((5, 1, page, D)), dtype) for _ in range(2))
    q = rnd(r.standard_normal((1, 1, D)), dtype)
    q[:, :, 0], k[:, :, :, 0] = 8, 0
    k[4, :, :, 0] = 22                                           # a score of 22 = 8 * 22 / sqrt(D)
    table = np.tile(np.arange(4, dtype=np.int32), 2 ** 25)[:width]
    table[-1] = 4
    got = mt.fused_ops.fused_paged_attention(dev(mt, q, dtype), dev(mt, k, dtype), dev(mt, v, dtype), i32(mt, table[None]), i32(mt, [0, 1]),
                                             i32(mt, [keys]), max_new=max_new).numpy()[0, 0]
    count = np.bincount(table, minlength=5).astype(np.float64).repeat(page).reshape(5, page)
    count[4, page - 5:] = 0
    s = np.einsum("d,pjd->pj", q[0, 0].astype(np.float64), k[:, 0].astype(np.float64)) / 8
    p = count * np.exp(s - s.max())
    p /= p.sum()
    assert 0.3 < p[4].sum() < 0.99
    want, A = np.einsum("pj,pjd->d", p, v[:, 0]), np.einsum("pj,pjd->d", p, np.abs(v[:, 0]))
    sums = 2 ** 26 / 592 * 8 if dtype == "float32" else 2 ** 24 / 444 * 4 if max_new == 1 else 2 ** 24 / 148 * 8
    allowed = (2 * sums * 2.0 ** -23 + 4 * U[dtype]) * A
    print(dtype, max_new, "error", np.abs(got - want).max(), "of", np.abs(want).max(), "allowed", allowed.min(), "last page", p[4].sum())
    assert (np.abs(got - want) <= allowed).all()
    no_device_flag(mt)


def test_the_most_rows_of_one_request(mt):
    """2^27 + 2^20 rows where a token was expected, in fp32: shares of them, weighed row by row, pass 64 bits. The last row sees
    the one key there is, all others see none. (All rows read one query; the output takes 35 GB.)"""
    torch = pytest.importorskip("torch")
    from mytorch_b200 import _lib
    from mytorch_b200.array import stream, synchronize
    rows, D = 2 ** 27 + 2 ** 20, 64
    out = torch.full((rows, D), float("nan"), device="cuda")
    pools = torch.arange(2 * 16 * D, device="cuda", dtype=torch.float32).view(2, 1, 16, D)
    ints = [torch.tensor(a, device="cuda", dtype=torch.int32) for a in ([[1, -1]], [0, rows], [1])]
    torch.cuda.synchronize()
    S = _lib.Strides3
    _lib.attn_paged(pools.data_ptr(), pools.data_ptr(), pools.data_ptr(), out.data_ptr(), S(0, D, 0), S(16 * D, 16 * D, D), S(0, D, D),
                    *[a.data_ptr() for a in ints], 1, 2, rows, 1, 1, 1, D, 16, 2, 0.125, _lib.F32, stream())
    synchronize()
    step = 1 << 22
    last, others = torch.equal(out[-1], pools[1, 0, 0]), all(not out[a:min(a + step, rows - 1)].any() for a in range(0, rows, step))
    del out
    torch.cuda.empty_cache()
    assert last and others


SCRATCH = """
import ctypes, torch
from mytorch_b200 import _lib, array
cu = ctypes.CDLL("libcuda.so.1")
def kept():
    pool, n = ctypes.c_void_p(), ctypes.c_uint64()
    assert cu.cuDeviceGetDefaultMemPool(ctypes.byref(pool), 0) == 0
    assert cu.cuMemPoolGetAttribute(pool, 4, ctypes.byref(n)) == 0          # the release threshold
    return n.value
x = torch.ones(10000, device="cuda")
out = torch.zeros(1, device="cuda")
torch.cuda.synchronize()
print(kept())
_lib.sum_f32(x.data_ptr(), _lib.F32, x.numel(), out.data_ptr(), array.stream())
print(kept())
q, o, pools = (torch.zeros(s, device="cuda", dtype=torch.float16) for s in ((40, 2, 64), (40, 2, 64), (100, 2, 16, 64)))
ints = [torch.tensor(a, device="cuda", dtype=torch.int32) for a in ([list(range(100))], [0, 40], [1600])]
torch.cuda.synchronize()
S = _lib.Strides3
for max_new in (1, 40):
    _lib.attn_paged(q.data_ptr(), pools.data_ptr(), pools.data_ptr(), o.data_ptr(), S(0, 64, 128), S(2048, 1024, 64), S(0, 64, 128),
                    *[a.data_ptr() for a in ints], 1, 100, 40, max_new, 2, 2, 64, 16, 100, 0.125, _lib.F16, array.stream())
    print(kept())
array.synchronize()
array.DeviceArray.empty((4,), "float32")
print(kept())
"""


def test_scratch_leaves_the_process_memory_pool_alone():
    """A program with buffers of its own keeps its device's default pool as it set it, whatever scratch the calls take; mt_malloc,
    which allocates from that pool, has it keep what is freed."""
    assert [int(n) for n in child(SCRATCH).split()] == [0, 0, 0, 0, 2 ** 64 - 1]


# Groups of query heads that fill a box of queries but none of outputs (64, 128), and that pass a tile of 128 rows or an item of 256.
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,D", [(64, 1, 64), (128, 2, 128), (128, 1, 64), (160, 1, 128), (320, 1, 64)])
def test_many_query_heads_for_one_of_the_cache(mt, dtype, heads, kv_heads, D):
    from tests.test_paged_gpu import Step, no_device_flag
    for batch in ([(1, 1), (129, 1), (300, 1)], [(40, 3), (1, 1), (0, 0), (150, 9), (5, 5), (64, 0), (257, 2)]):
        Step(batch, heads, kv_heads, D, 16, dtype).check(mt, max_new=max(m for _, m in batch))
    Step([(70, 6), (33, 2)], heads, kv_heads, D, 7, dtype, pad=0).check(mt)
    no_device_flag(mt)


def test_nan_at_the_start_of_a_long_cache(mt):
    """A value that is NaN makes 256 rows of 140000 keys be computed again one by one, for 2.6 s, beside 295 requests that are finite: longer
    than any wait within the kernel may last, so nothing may wait for it, and no row is lost: the others have the bits that they have
    without it. The same rows' other columns, two ways: sums of fp16 weights (off by 2^-11) against fp32 ones, both of 140000 terms
    in fp32 (140008 * 2^-24 of sum_j p_j |v_j| < 1 at most, in output and weights' sum), rounded once."""
    from tests.test_ops_gpu import dev
    from tests.test_paged_gpu import device_flag, i32
    N, D, page, R, new = 140000, 64, 128, 296, 256
    n = -(-N // page)
    r = np.random.default_rng(0)
    k, v = (r.standard_normal((n + 1, 1, page, D)).astype(np.float16) for _ in range(2))
    k[n], v[n] = k[0], v[0]
    v[n, 0, 3, 5] = np.nan
    Q, K, V = (dev(mt, a, "float16") for a in (r.standard_normal((R * new, 1, D)), k, v))
    tables = np.tile(np.arange(n), (R, 1))

    def ask():
        return mt.fused_ops.fused_paged_attention(Q, K, V, i32(mt, tables), i32(mt, np.arange(R + 1) * new), i32(mt, [N] * R),
                                                  max_new=new).numpy()[:, 0]
    clean = ask()
    tables[0, 0] = n                                             # for request 0 alone
    got = ask()
    assert device_flag(mt) == 0 and np.isfinite(clean).all()
    assert np.array_equal(got[new:], clean[new:])
    assert np.isnan(got[:new, 5]).all()
    a, b = (np.delete(x[:new], 5, 1).astype(np.float64) for x in (got, clean))
    assert (np.abs(a - b) <= 3 * 2.0 ** -11 + 4 * (N + 8) * 2.0 ** -24).all()
