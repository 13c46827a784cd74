"""The paged cache as programs use it: tables, appends and attention of step after step with requests that join
and leave, both models' forwards over it against their contiguous caches, generate() with prompts of different
lengths, and a step captured into a CUDA graph."""
import ctypes as C

import numpy as np
import pytest

from tests.test_infer_gpu import cache_of, models
from tests.test_ops_gpu import DTYPES, TOL, close, dev, no_device_flag, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    import mytorch_b200 as m
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 2, 64, 16), (5, 1, 128, 24), (2, 2, 64, 7)])
def test_requests_come_and_go(mt, dtype, heads, kv_heads, D, page):
    """Every request's rows are attention over its own history, whatever pages it got and whoever had them before."""
    r = np.random.default_rng(page)
    cache = mt.PagedKVCache(num_pages=60, page_size=page, num_heads=kv_heads, head_dim=D, num_layers=2, max_requests=4, max_len=60 * page)
    history = [[np.zeros((2, 2, 0, kv_heads, D), np.float32)] for _ in range(4)]
    plan = [([40, 0, 3], []), ([1, 70, 1, 0], [0]), ([33, 1, 1, 5], []), ([1, 1, 1, 1], [1, 3]), ([2, 90, 0, 20], []), ([1, 1, 1, 1], [2])]
    for fresh, over in plan:
        cache.begin(fresh)
        n = sum(fresh)
        first = np.concatenate([[0], np.cumsum(fresh)])
        for layer in range(2):
            k, v, q = (rnd(r.standard_normal((n, h, D)), dtype) for h in (kv_heads, kv_heads, heads))
            cache.update(dev(mt, k, dtype), dev(mt, v, dtype), layer)
            got = cache.attend(dev(mt, q, dtype), layer).numpy()
            for i, m in enumerate(fresh):
                rows = slice(first[i], first[i + 1])
                if layer == 0:
                    history[i].append(np.zeros((2, 2, m, kv_heads, D), np.float32))
                history[i][-1][layer] = k[rows], v[rows]
                kk, vv = (np.concatenate([h[layer, w] for h in history[i]]).astype(np.float64).repeat(heads // kv_heads, 1) for w in (0, 1))
                s = np.einsum("mhd,nhd->hmn", q[rows].astype(np.float64), kk) * D ** -0.5
                s = np.where(np.arange(len(kk)) <= np.arange(len(kk) - m, len(kk))[:, None], s, -np.inf)
                p = np.exp(s - s.max(-1, keepdims=True)) if m else s
                want = np.einsum("hmn,nhd->mhd", p / p.sum(-1, keepdims=True) if m else p, vv)
                if m:
                    close(got[rows], want, TOL[dtype], f"request {i}")
        assert np.array_equal(cache.kv_len.numpy(), cache.lengths)
        if over:
            cache.release(over)
            for i in over:
                history[i] = history[i][:1]
    no_device_flag(mt)
    used = [t for row, n in zip(cache.tables.numpy(), cache.lengths) for t in row[:-(-n // page)]]
    free = cache.free_pages.numpy()[:60 - len(used)]
    assert sorted(used + list(free)) == list(range(60))                      # every page is in one place


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,heads,kv_heads,D,bias", [("gpt2", 2, 2, 64, True), ("nanochat", 4, 2, 64, False), ("nanochat", 5, 1, 128, True)])
def test_models_over_pages(mt, dtype, kind, heads, kv_heads, D, bias):
    """Prompts of different lengths together, then tokens (several at once for one request): the logits of each request alone."""
    model = models(mt, kind, dtype, heads, kv_heads, D, bias)
    r = np.random.default_rng(7)
    lens, steps = [5, 70, 33], [[1, 1, 1], [1, 3, 1], [0, 1, 1]]
    ids = [r.integers(0, 200, n + 5).astype(np.int32) for n in lens]
    cache = mt.PagedKVCache(40, 16, kv_heads, D, 2, 3, 160)
    alone = [cache_of(mt, model, kind, 1) for _ in ids]
    at = [0, 0, 0]
    with mt.no_grad():
        for fresh in [lens] + steps:
            new = [a[i:i + n] for a, i, n in zip(ids, at, fresh)]
            logits, _ = model(mt.Tensor(np.concatenate(new)[None]), cache=cache.begin(fresh))
            assert logits.shape == (3, 1, logits.shape[2])
            for i, x in enumerate(new):
                at[i] += len(x)
                if len(x):
                    # the contiguous GPT-2 cache lets several new tokens see each other, so they go in one by one
                    for part in ([x] if at[i] == len(x) else np.split(x, len(x))):
                        want = model(mt.Tensor(part[None]), cache=alone[i])[0]
                    close(logits.numpy()[i, 0], want.numpy()[0, -1], 2 * TOL[dtype], f"request {i}")
    no_device_flag(mt)


@pytest.mark.parametrize("kind", ["gpt2", "nanochat"])
def test_generate_from_prompts_of_different_lengths(mt, kind):
    model = models(mt, kind, "float32", 2, 2, 64, False)
    r = np.random.default_rng(9)
    prompts = [r.integers(0, 200, n).astype(np.int32) for n in (3, 40, 17)]
    got = model.generate(prompts, 6, temperature=0)
    for p, g in zip(prompts, got):
        assert np.array_equal(g, model.generate(p[None], 6, temperature=0)[0])
    drawn = model.generate(prompts, 4, temperature=0.8, top_k=5, seed=1)
    assert [len(g) for g in drawn] == [7, 44, 21] and all((0 <= g).all() and (g < 203).all() for g in drawn)


def test_refusals(mt):
    model = models(mt, "nanochat", "float16", 4, 2, 64, False)
    cache = mt.PagedKVCache(4, 16, 2, 64, 2, 2, 64)
    ids = mt.Tensor(np.zeros((1, 5), np.int32))
    with mt.no_grad():
        with pytest.raises(ValueError):
            model(ids, cache=cache)                              # begin() was not called
        for bad in ([1, 1, 1], [-1], [1.0, -2.0]):
            with pytest.raises(ValueError):
                cache.begin(bad)
        with pytest.raises(RuntimeError):
            cache.begin([65])                                    # more than a request may hold
        with pytest.raises(RuntimeError):
            cache.begin([33, 33])                                # more than there are pages
        cache.begin([4])
        with pytest.raises(ValueError):
            model(ids, cache=cache)                              # 5 ids for 4 announced tokens
        for other in (mt.PagedKVCache(4, 16, 4, 64, 2, 2, 64), mt.PagedKVCache(4, 16, 2, 64, 3, 2, 64), mt.PagedKVCache(20, 16, 2, 64, 2, 2, 161)):
            with pytest.raises(ValueError):
                model(ids, cache=other.begin([5]))
        with pytest.raises(ValueError):
            model(mt.Tensor(np.zeros((1, 4), np.int32)), mt.Tensor(np.zeros((1, 4), np.int32)), cache=cache)
        with pytest.raises(ValueError):
            model.generate([[1, 2], []], 3)
    for p in model.parameters():
        p.requires_grad = True
    with pytest.raises(NotImplementedError):
        model(mt.Tensor(np.zeros((1, 4), np.int32)), cache=cache)
    for bad in (dict(head_dim=96), dict(num_pages=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            mt.PagedKVCache(**{**dict(num_pages=4, page_size=16, num_heads=2, head_dim=64, num_layers=2, max_requests=2, max_len=64), **bad})


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("max_new", [1, 40])
def test_a_captured_step(mt, dtype, max_new):
    """Tables, append and attention captured once and replayed with other lengths: what a program with static
    buffers does. Two captured graphs have scratch of their own: replayed on two streams at once they do not disturb each other."""
    torch = pytest.importorskip("torch")
    from mytorch_b200 import array, fused_ops as K
    H, Hk, D, page, R, rows = 4, 2, 64, 16, 3, 3 * max_new
    r = np.random.default_rng(max_new)
    ints = lambda a: mt.DeviceArray.from_numpy(np.asarray(a, np.int32), "int32")

    def world(seed):
        g = np.random.default_rng(seed)
        pools = [dev(mt, rnd(g.standard_normal((40, Hk, page, D)), dtype), dtype) for _ in range(2)]
        new = [dev(mt, rnd(g.standard_normal((rows, h, D)), dtype), dtype) for h in (Hk, Hk, H)]
        perm = g.permutation(40).astype(np.int32)
        tables = np.full((R, 12), -1, np.int32)
        tables[:, :4] = perm[:12].reshape(3, 4)
        return dict(pools=pools, new=new, held=ints([0, 0, 0]), fresh=ints([0, 0, 0]), tables=ints(tables), free=ints(np.r_[perm[12:], np.full(12, -1)]),
                    n_free=ints([28]), out=[ints(np.zeros(n)) for n in (R + 1, R, rows, rows, 1)], o=dev(mt, np.zeros((rows, H, D)), dtype), start=tables)

    def step(w):
        K.fused_paged_tables(w["held"], w["fresh"], w["tables"], w["free"], w["n_free"], page, out=w["out"])
        K.fused_paged_append(w["new"][0], w["new"][1], *w["pools"], w["out"][3])
        K.fused_paged_attention(w["new"][2], *w["pools"], w["tables"], w["out"][0], w["out"][1], max_new=max_new, out=w["o"])

    def lengths(w, held, fresh):
        w["held"].set_from_numpy(np.array(held, np.int32))
        w["fresh"].set_from_numpy(np.array(fresh, np.int32))
        w["tables"].set_from_numpy(w["start"])
        w["o"].zero_()
        array.synchronize()

    worlds, graphs, before = [world(1), world(2)], [], array.stream()
    for w in worlds:                                             # first calls look up device addresses and raise limits
        lengths(w, [50, 61, 1], [1, max_new, 1])
        step(w)
    array.synchronize()
    streams = [torch.cuda.Stream() for _ in worlds]
    try:
        for w, s in zip(worlds, streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s, capture_error_mode="relaxed"):
                array.set_stream(C.c_void_p(torch.cuda.current_stream().cuda_stream))
                step(w)
            graphs.append(g)
    finally:
        array.set_stream(before)
    cases = [([50, 61, 1], [1, max_new, 1]), ([0, 63, 17], [max_new, 0, max_new]), ([64, 0, 33], [1, 1, 1])]
    for held, fresh in cases:
        want = []
        for w in worlds:
            lengths(w, held, fresh)
            step(w)
            want.append([a.numpy() for a in [w["o"], w["tables"], *w["out"], *w["pools"]]])
            lengths(w, held, fresh)
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for w, x in zip(worlds, want):
            for a, b in zip([w["o"], w["tables"], *w["out"], *w["pools"]], x):
                assert np.array_equal(a.numpy(), b)
    del graphs
    no_device_flag(mt)
