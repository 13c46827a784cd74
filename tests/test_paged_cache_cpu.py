"""The host side of the paged cache: what begin(), update(), release() and generate() announce and refuse. Device arrays
are NumPy arrays here and the library's calls are done by hand, so these run without a GPU."""
import numpy as np
import pytest


class Array:
    """A device array's shape, type and contents on the host."""

    def __init__(self, a):
        self.a = np.asarray(a)

    shape = property(lambda self: self.a.shape)
    dtype = property(lambda self: str(self.a.dtype))
    size = property(lambda self: self.a.size)

    @classmethod
    def empty(cls, shape, dtype="float32"):
        return cls(np.zeros(shape, dtype))

    zeros = empty

    @classmethod
    def from_numpy(cls, a, dtype=None):
        return cls(np.array(a, dtype))

    def numpy(self):
        return self.a.copy()

    def reshape(self, *shape):
        return Array(self.a.reshape(*shape))

    def rows(self, a, b):
        return Array(self.a[a:b])

    def zero_(self):
        self.a[...] = 0


def tables(held, fresh, table, free, n_free, page, out):
    """fused_paged_tables, one page after the other."""
    starts, kv_len, position, slot, left = (o.a for o in out)
    n = int(n_free.a[0])
    starts[0] = 0
    for r, (h, f) in enumerate(zip(held.a, fresh.a)):
        for at in range(-(-h // page), -(-(h + f) // page)):
            n -= 1
            table.a[r, at] = free.a[n]
        starts[r + 1], kv_len[r] = starts[r] + f, h + f
        j = np.arange(h, h + f)
        position[starts[r]:starts[r + 1]] = j
        slot[starts[r]:starts[r + 1]] = table.a[r, j // page] * page + j % page
    left[0] = n


def release(done, table, kv_len, free, n_free, page):
    for r in np.flatnonzero(done.a):
        for at in range(-(-kv_len.a[r] // page)):
            free.a[n_free.a[0]] = table.a[r, at]
            n_free.a[0] += 1
            table.a[r, at] = -1
        kv_len.a[r] = 0


def append(k, v, k_pages, v_pages, slot, strides=None):
    page = k_pages.shape[2]
    for i, s in enumerate(slot.a):
        k_pages.a[s // page, :, s % page], v_pages.a[s // page, :, s % page] = k.a[i], v.a[i]


@pytest.fixture()
def paged(monkeypatch):
    from mytorch_b200 import paged
    monkeypatch.setattr(paged, "DeviceArray", Array)
    monkeypatch.setattr(paged.K, "fused_paged_tables", tables)
    monkeypatch.setattr(paged.K, "fused_paged_release", release)
    monkeypatch.setattr(paged.K, "fused_paged_append", append)
    return paged


def a_cache(paged, **how):
    return paged.PagedKVCache(**{**dict(num_pages=12, page_size=4, num_heads=1, head_dim=64, num_layers=2, max_requests=3, max_len=16), **how})


def fill(cache, value=1.0):
    """The step's rows of every layer."""
    for layer in range(cache.shape[0]):
        cache.update(*(Array(np.full((cache.rows, 1, 64), value, np.float32)) for _ in range(2)), layer)


def step(cache, fresh):
    cache.begin(fresh)
    fill(cache)
    return cache


def test_one_row_of_logits_for_every_count_given(paged):
    """Counts that are filled up with zeros to the same step still ask for another number of rows."""
    cache = a_cache(paged)
    assert list(step(cache, [1, 1]).last_rows.a) == [0, 1]
    assert len(step(cache, [1, 1, 0]).last_rows.a) == 3
    assert len(step(cache, [1, 1]).last_rows.a) == 2
    assert len(step(cache, [1]).last_rows.a) == 1
    assert len(step(cache, [1, 0]).last_rows.a) == 2
    assert list(cache.lengths) == [5, 3, 0] and list(cache.kv_len.a) == [5, 3, 0]


def test_requests_without_new_tokens_have_no_logits(paged):
    cache = a_cache(paged, max_requests=6)
    for fresh in ([5, 0, 3], [0, 1, 1], [1, 0, 0, 2, 0], [0, 0, 0, 0, 0, 1], [1, 1], [0, 1, 0]):
        step(cache, fresh)
        got = cache.clear_idle(Array(np.full((len(fresh), 1, 7), 3.0)))
        assert (got.a[:, 0] == np.where(np.array(fresh)[:, None] > 0, 3.0, 0.0)).all(), fresh


@pytest.mark.parametrize("layer", [2, -1, 5])
def test_layers_that_the_cache_does_not_have(paged, layer, monkeypatch):
    """Such a layer's pools would lie outside the memory of the cache: nothing is queued for it."""
    cache = step(a_cache(paged), [3])
    for name in ("fused_paged_append", "fused_paged_attention"):
        monkeypatch.setattr(paged.K, name, lambda *a, **k: pytest.fail("reached the library"))
    rows = Array(np.zeros((3, 1, 64), np.float32))
    for call in (lambda: cache.update(rows, rows, layer), lambda: cache.attend(rows, layer)):
        with pytest.raises(IndexError):
            call()


def test_calls_before_there_is_anything_to_work_on(paged):
    cache, rows = a_cache(paged), Array(np.zeros((3, 1, 64), np.float32))
    with pytest.raises(RuntimeError):
        cache.update(rows, rows, 0)                              # no step was begun
    cache.begin([3])
    with pytest.raises(RuntimeError):
        cache.attend(rows, 0)                                    # no row was ever appended


@pytest.mark.parametrize("rows", [2, 4])
def test_as_many_queries_as_the_step_has_rows(paged, rows, monkeypatch):
    """More would leave rows of the result as they were allocated, fewer would leave out rows of requests."""
    cache = step(a_cache(paged), [2, 1])
    monkeypatch.setattr(paged.K, "fused_paged_attention", lambda *a, **k: pytest.fail("reached the library"))
    with pytest.raises(ValueError):
        cache.attend(Array(np.zeros((rows, 1, 64), np.float32)), 0)


def test_a_refused_first_update_leaves_no_pools_behind(paged, monkeypatch):
    """The pools have the type of the first rows that are taken, not of some that were refused."""
    def refuse(*a, **k):
        raise TypeError
    cache = a_cache(paged).begin([3])
    with monkeypatch.context() as m:
        m.setattr(paged.K, "fused_paged_append", refuse)
        with pytest.raises(TypeError):
            cache.update(*(Array(np.zeros((3, 1, 64), np.int32)) for _ in range(2)), 0)
    fill(cache)
    assert cache.k_pages.dtype == cache.v_pages.dtype == "float32"


@pytest.mark.parametrize("lengths,new", [([3, 6], 3), ([8, 1, 4], 1), ([16, 15], 1), ([9, 1], 8)])
def test_generate_asks_for_no_more_than_it_feeds(paged, lengths, new):
    """The last token is drawn and never fed: a request holds one row less than its tokens."""
    made = []

    def new_cache(requests, longest, rows):
        made.append(paged.cache_for(2, 1, 64, page_size=4)(requests, longest, rows))
        return made[0]

    def model(ids, cache):
        cache.check(ids.shape, 2, 1, 64, 16)
        fill(cache)
        return Array(np.zeros((len(lengths), 1, 5), np.float32))
    out = paged.generate(model, [np.arange(n) for n in lengths], new, lambda logits: Array(np.full(len(lengths), 9, np.int32)), new_cache)
    assert [list(o) for o in out] == [list(range(n)) + [9] * new for n in lengths]
    held = np.array(lengths) + new - 1
    assert list(made[0].lengths) == list(held) and made[0].max_len == held.max() and made[0].shape[1] == made[0].pages_used()


def same_state(a, b):
    """What later steps depend on: lengths, free pages in order, and the tables' entries in use."""
    assert list(a.lengths) == list(b.lengths) and list(a.kv_len.a) == list(b.kv_len.a)
    n = a._n_free.a[0]
    assert n == b._n_free.a[0] and list(a.free_pages.a[:n]) == list(b.free_pages.a[:n])
    for r, held in enumerate(a.lengths):
        used = -(-held // a.page_size)
        assert list(a.tables.a[r, :used]) == list(b.tables.a[r, :used])


def test_a_step_whose_rows_were_not_appended(paged):
    """Its rows would count as held and be read as keys and values: the next step is refused until they are there, or taken back."""
    cache, other = step(a_cache(paged), [3, 5]), step(a_cache(paged), [3, 5])
    cache.begin([6, 2])
    with pytest.raises(ValueError):
        cache.check((1, 7), 2, 1, 64, 16)                        # a forward that was refused
    for appended in range(2):                                    # none of the two layers, one of them
        for fresh in ([6, 2], [1], [0]):
            with pytest.raises(RuntimeError):
                cache.begin(fresh)
        cache.update(*(Array(np.ones((8, 1, 64), np.float32)) for _ in range(2)), appended)
    cache.begin([1, 0, 4]).cancel()                              # both are there: the next one, which is taken back
    same_state(cache, step(other, [6, 2]))
    rows = Array(np.ones((5, 1, 64), np.float32))
    with pytest.raises(RuntimeError):
        cache.update(rows, rows, 0)                              # a step that was taken back has no slots
    same_state(step(cache, [2, 1]), step(other, [2, 1]))
    with pytest.raises(RuntimeError):
        cache.cancel()                                           # its rows are there


def test_a_step_taken_back_half_way(paged):
    cache, other = step(a_cache(paged), [3, 5]), step(a_cache(paged), [3, 5])
    cache.begin([9, 2])
    cache.update(*(Array(np.ones((11, 1, 64), np.float32)) for _ in range(2)), 1)
    cache.cancel()
    same_state(cache, other)
    for c in (cache, other):
        step(c, [1, 7, 2])
        c.release([1])
        step(c, [4, 3])
    same_state(cache, other)


def test_steps_without_tokens_leave_nothing_open(paged):
    cache = a_cache(paged)
    cache.begin([0, 0]).begin([]).begin([1])
    assert list(cache.lengths) == [1, 0, 0]


def test_release_within_a_step(paged):
    """Requests that a forward under way brings tokens for cannot go; after others went, the step can no longer be taken back."""
    cache, other = step(a_cache(paged), [3, 5]), step(a_cache(paged), [3, 5])
    cache.begin([0, 2])
    cache.update(*(Array(np.ones((2, 1, 64), np.float32)) for _ in range(2)), 0)
    with pytest.raises(RuntimeError):
        cache.release([1])
    assert list(cache.lengths) == [3, 7, 0]
    cache.release([0])
    with pytest.raises(RuntimeError):
        cache.cancel()
    fill(cache)
    other = step(other, [0, 2])
    other.release([0])
    same_state(cache, other)
    cache.release([1])
    assert sorted(cache.free_pages.a) == list(range(12))


def test_a_program_with_pools_of_its_own(paged):
    """One that takes tables and slots from the cache and appends by itself: steps follow each other, requests go when they like; a
    request that went in a step leaves no step behind that a forward could run."""
    cache, other = a_cache(paged), a_cache(paged)
    for fresh, over in (([3, 5], []), ([1, 1, 2], [1]), ([2, 4], [0, 2]), ([0, 1], [])):
        cache.begin(fresh)
        assert len(cache.slot.a) == sum(fresh)
        step(other, fresh)
        for c in (cache, other):
            c.release(over)
        same_state(cache, other)
    cache.release([1])
    rows = Array(np.zeros((1, 1, 64), np.float32))
    with pytest.raises(RuntimeError):
        cache.update(rows, rows, 0)
    with pytest.raises(RuntimeError):
        cache.attend(rows, 0)
    with pytest.raises(ValueError):
        cache.check((1, 1), 2, 1, 64, 16)
    other.release([1])
    same_state(step(cache, [2]), step(other, [2]))


def test_places_and_counts_that_are_none(paged):
    cache = step(a_cache(paged), [3, 5, 1])
    for bad in ([-1], [0, -3], [3], -1, 3):
        with pytest.raises(IndexError):
            cache.release(bad)
    for bad in ([1.5], [True, False, True], ["1"], [float("nan")]):
        with pytest.raises(ValueError):
            cache.release(bad)
    for bad in ([5.9], [float("nan")], [float("inf")], [2.0, 0.5], ["2"], [2 ** 63]):
        with pytest.raises(ValueError):
            cache.begin(bad)
    assert list(cache.lengths) == [3, 5, 1] and list(cache.kv_len.a) == [3, 5, 1]
    step(cache, [2.0, 1.0])                                      # whole numbers, whatever their type
    step(cache, np.array([1, 1], np.uint8))
    step(cache, [True, False])
    cache.release(())
    cache.release(np.array([0.0, 2.0]))
    cache.release(1)
    assert list(cache.lengths) == [0, 0, 0] and sorted(cache.free_pages.a) == list(range(12))


def test_a_refused_generate_leaves_the_model_as_it_was():
    """Prompts of different lengths, one of them empty: the model trains on afterwards."""
    from types import SimpleNamespace
    from mytorch_b200.nanochat_gpt import GPT
    model = SimpleNamespace(training=True, config=SimpleNamespace(num_blocks=2, num_kv_heads=1, embed_dim=64, num_q_heads=1))
    model.eval = lambda: setattr(model, "training", False)
    model.train = lambda: setattr(model, "training", True)
    with pytest.raises(ValueError):
        GPT.generate(model, [[1, 2], []], 3)
    assert model.training


def test_a_step_that_the_library_refused(paged, monkeypatch):
    """Its positions and slots were never written: no forward can run it, and the cache is as before."""
    def refuse(*a, **k):
        raise RuntimeError("refused")
    cache, other = step(a_cache(paged), [3, 5]), step(a_cache(paged), [3, 5])
    for fresh in ([1, 1], [3, 5]):                               # with arrays made anew, and with those of the step before
        with monkeypatch.context() as m:
            m.setattr(paged.K, "fused_paged_tables", refuse)
            with pytest.raises(RuntimeError):
                cache.begin(fresh)
        with pytest.raises(ValueError):
            cache.check((1, sum(fresh)), 2, 1, 64, 16)
        with pytest.raises(RuntimeError):
            fill(cache)
        same_state(cache, other)
    same_state(step(cache, [1, 1]), step(other, [1, 1]))
