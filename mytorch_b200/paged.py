"""A key/value cache in pages, for requests of different lengths that come and go (the counterpart of
nanochat_gpt.KVCache and gpt2.Cache, which hold one length for a whole batch).

Both models' forward takes one as `cache`, with the new tokens of all requests packed one behind the other:

    cache = PagedKVCache(num_pages=512, page_size=16, num_heads=kv_heads, head_dim=D, num_layers=L, max_requests=8, max_len=2048)
    cache.begin([5, 0, 9])                       # 5 new tokens for request 0, 9 for request 2
    logits, cache = model(packed_ids, cache=cache)   # ids [1, 14] -> logits [3, 1, V] behind each request's last token, 0 for request 1
    cache.release([0])                           # request 0 is over; its pages are free again

Tables, slots and positions are computed on the device (fused_ops.fused_paged_tables); the host keeps the
lengths too, so that a step that does not fit is refused before anything is launched."""
import numpy as np

from . import _lib, fused_ops as K
from .array import DeviceArray, stream


def _whole(what, values, kinds="iuf"):
    """Whole numbers of any type as int64; anything else is refused rather than rounded."""
    a = np.asarray(values).reshape(-1)
    if a.size and (a.dtype.kind not in kinds or not (np.abs(a) < 2 ** 31).all() or (a != np.floor(a)).any()):
        raise ValueError(f"{what} are whole numbers below 2^31, got {values}")
    return a.astype(np.int64)


class PagedKVCache:
    def __init__(self, num_pages, page_size, num_heads, head_dim, num_layers, max_requests, max_len):
        if min(num_pages, page_size, num_heads, num_layers, max_requests, max_len) < 1:
            raise ValueError("every size of a paged cache is at least 1")
        if head_dim not in (64, 128):
            raise ValueError(f"attention over pages is built for heads of 64 and 128, got {head_dim}")
        self.shape = (num_layers, num_pages, num_heads, page_size, head_dim)
        self.page_size, self.max_len = page_size, max_len
        self.k_pages = self.v_pages = None                       # made with the first update, in its dtype
        width = -(-max_len // page_size)
        ints = lambda a: DeviceArray.from_numpy(np.asarray(a, np.int32), "int32")
        self.tables = ints(np.full((max_requests, width), -1))
        self.free_pages = ints(np.arange(num_pages)[::-1])       # taken from the end: page 0 first
        self._n_free, self._next_free = ints([num_pages]), ints([0])
        self._held, self._kv_len = ints(np.zeros(max_requests)), ints(np.zeros(max_requests))
        self.starts = self.position = self.slot = None
        self.lengths = np.zeros(max_requests, np.int64)          # the host's copy of the lengths
        self._fresh, self._fresh_dev = None, None
        # The step's layers without its rows; whether a forward of it began; whether requests went since it began.
        self._missing, self._running, self._released = set(), False, False

    @property
    def kv_len(self):
        """Rows of every request on the device, this step's among them."""
        return self._held

    def pages_used(self, lengths=None):
        return int((-(-(self.lengths if lengths is None else lengths) // self.page_size)).sum())

    def begin(self, fresh):
        """Starts a step with fresh[r] new tokens for request r (shorter lists are filled up with zeros). From here on they count as
        held, so after a forward that was refused or failed it is run again, or the step taken back by cancel(), before the next begins."""
        if self._running and self._missing:
            raise RuntimeError(f"the step before is without its rows in {len(self._missing)} of {self.shape[0]} layers: run its forward, or cancel() it")
        counts = np.zeros(len(self.lengths), np.int64)
        fresh = _whole("counts of new tokens", fresh, "iufb")
        if len(fresh) > len(counts) or (fresh < 0).any():
            raise ValueError(f"a step takes up to {len(counts)} counts of new tokens, none negative; got {fresh.tolist()}")
        counts[:len(fresh)] = fresh
        after = self.lengths + counts
        if (after > self.max_len).any():
            raise RuntimeError(f"request {int(after.argmax())} would hold {int(after.max())} tokens of at most {self.max_len}")
        if self.pages_used(after) > self.shape[1]:
            raise RuntimeError(f"{self.pages_used(after)} pages are needed and {self.shape[1]} exist: release a request first")
        # A decoding step asks for the same as the one before. How many counts were given belongs to it: there are as many last rows.
        if self._fresh is None or not np.array_equal(self._fresh, fresh):
            self._end()                                          # until everything below is made
            n = int(counts.sum())
            self._fresh_dev = DeviceArray.from_numpy(counts, "int32")
            self.starts = DeviceArray.empty((len(counts) + 1,), "int32")
            self.position, self.slot = DeviceArray.empty((n,), "int32"), DeviceArray.empty((n,), "int32")
            self.last_rows = DeviceArray.from_numpy(np.maximum(np.cumsum(counts)[:max(1, len(fresh))] - 1, 0), "int32")
            self.max_new, self.rows = int(counts.max()), n
            self._idle = np.flatnonzero(np.diff(np.r_[0, fresh == 0, 0])).reshape(-1, 2).tolist()     # [first, end) of requests without new tokens
            self._fresh = fresh.copy()
        try:
            K.fused_paged_tables(self._held, self._fresh_dev, self.tables, self.free_pages, self._n_free, self.page_size,
                                 out=(self.starts, self._kv_len, self.position, self.slot, self._next_free))
        except Exception:
            self._end()                                          # nothing was written there
            raise
        self._held, self._kv_len = self._kv_len, self._held
        self._n_free, self._next_free = self._next_free, self._n_free
        self.lengths = after
        self._missing, self._running, self._released = set(range(self.shape[0]) if self.rows else ()), False, False
        return self

    def cancel(self):
        """Takes the step back whose rows are not in every layer yet: lengths and free pages are as before its begin()."""
        if not self._missing or self.slot is None:
            raise RuntimeError("there is no step to take back: none was begun, or its rows are in every layer")
        if self._released:
            raise RuntimeError("requests were released since this step began: it can no longer be taken back")
        self._held, self._kv_len = self._kv_len, self._held
        self._n_free, self._next_free = self._next_free, self._n_free
        self.lengths[:len(self._fresh)] -= self._fresh
        self._end()

    def _end(self):
        """Nothing of this step can be asked for any more."""
        self.starts = self.position = self.slot = self._fresh = None
        self._missing, self._running = set(), False

    def release(self, requests):
        """These requests are over: their pages are free and their places may be used by new ones."""
        done = np.zeros(len(self.lengths), np.int32)
        places = _whole("requests", requests)
        if ((places < 0) | (places >= len(done))).any():
            raise IndexError(f"the requests are 0 to {len(done) - 1}, got {places.tolist()}")
        done[places] = 1
        if self._missing:
            if done[:len(self._fresh)][self._fresh > 0].any():   # with tokens in this step
                if self._running:
                    raise RuntimeError("a request cannot go while a forward brings tokens for it: run it to its end, or cancel() the step")
                self._end()
            self._released = True
        K.fused_paged_release(DeviceArray.from_numpy(done, "int32"), self.tables, self._held, self.free_pages, self._n_free, self.page_size)
        self.lengths[done != 0] = 0

    def _layer(self, pools, layer_idx):
        if not 0 <= layer_idx < self.shape[0]:
            raise IndexError(f"layer {layer_idx} of {self.shape[0]}")
        return pools.rows(layer_idx, layer_idx + 1).reshape(self.shape[1:])

    def update(self, k, v, layer_idx, strides=None):
        """The step's new keys and values [rows, heads, head_dim] of one layer (`strides`: two Strides3 of a view)."""
        if self.slot is None:
            raise RuntimeError("no step was begun")
        pools = (self.k_pages, self.v_pages) if self.k_pages is not None else [DeviceArray.zeros(self.shape, k.dtype) for _ in range(2)]
        K.fused_paged_append(k, v, *(self._layer(p, layer_idx) for p in pools), self.slot, strides)
        self.k_pages, self.v_pages = pools                       # the first rows that are taken settle the type
        self._running = True
        self._missing.discard(layer_idx)

    def attend(self, q, layer_idx, strides=None):
        """Causal attention of the step's rows q [rows, query heads, head_dim] over one layer's pages."""
        if self.k_pages is None or self.slot is None:
            raise RuntimeError("no row of this step was appended yet")
        if q.shape[0] != self.rows:
            raise ValueError(f"begin() announced {self.rows} tokens, got queries of {q.shape[0]}")
        out = DeviceArray.empty(q.shape, q.dtype)                # begin()'s rows are exactly the requests' rows
        return K.fused_paged_attention(q, self._layer(self.k_pages, layer_idx), self._layer(self.v_pages, layer_idx), self.tables,
                                       self.starts, self._held, max_new=self.max_new, out=out, strides=strides)

    def clear_idle(self, logits):
        """Logits [requests, ...]: zeros for the requests that have no new token, whose last row is another request's."""
        for first, end in self._idle:
            logits.rows(first, end).zero_()
        return logits

    def check(self, ids_shape, num_layers, num_heads, head_dim, max_positions):
        """Refuses a model or ids that this cache and step are not for. The step's forward begins here."""
        self._running = True
        if self.starts is None or tuple(ids_shape) != (1, self.rows) or self.rows == 0:
            raise ValueError(f"begin() announced {0 if self.starts is None else self.rows} tokens; ids of shape (1, that many) are expected, got {tuple(ids_shape)}")
        L, _, H, _, D = self.shape
        if (L, H, D) != (num_layers, num_heads, head_dim):
            raise ValueError(f"the cache holds {L} layers of {H} heads of {D}, the model has {num_layers} of {num_heads} of {head_dim}")
        if self.max_len > max_positions:
            raise ValueError(f"the cache allows {self.max_len} tokens per request, the model has {max_positions} positions")


def generate(model, prompts, max_new_tokens, pick, new_cache):
    """Prompts of different lengths, each followed by max_new_tokens tokens: [ids + tokens per prompt].
    pick(logits) -> next token per request, int32 [requests] on the device; new_cache(requests, the longest one's rows, every one's rows)."""
    prompts = [np.asarray(p, np.int32).reshape(-1) for p in prompts]
    if any(len(p) == 0 for p in prompts):
        raise ValueError("every prompt needs a token")
    if max_new_tokens < 1 or not prompts:
        return prompts
    R = len(prompts)
    rows = [len(p) + max_new_tokens - 1 for p in prompts]        # the last token is drawn and not fed
    cache = new_cache(R, max(rows), rows)
    feed, fresh, out = DeviceArray.from_numpy(np.concatenate(prompts), "int32"), [len(p) for p in prompts], []
    for i in range(max_new_tokens):
        logits = model(feed.reshape(1, -1), cache.begin(fresh))
        feed, fresh = pick(logits), [1] * R
        out.append(feed)
    tokens = np.stack([t.numpy() for t in out], 1)
    return [np.concatenate([p, t]) for p, t in zip(prompts, tokens)]


def is_ragged(input_ids):
    """Prompts as a list or tuple of sequences that are not all equally long."""
    return isinstance(input_ids, (list, tuple)) and len(input_ids) > 0 and all(np.ndim(p) == 1 for p in input_ids) \
        and len({len(p) for p in input_ids}) > 1


def sampler(temperature, top_k, rng):
    """How generate() picks: the arg-max on the device for temperature 0, else a draw per request on the host."""
    def pick(logits):
        R, _, V = logits.shape
        if temperature == 0:
            nxt, out = DeviceArray.empty((R,), "int32"), DeviceArray.empty((R,), "int32")
            _lib.argmax_rows(logits.ptr, nxt.ptr, out.ptr, R, V, 1, logits.code, stream())
            return nxt
        last = logits.numpy()[:, -1, :].astype(np.float64) / temperature
        if top_k is not None:
            kth = np.sort(last, -1)[:, -top_k][:, None]
            last = np.where(last < kth, -np.inf, last)
        p = np.exp(last - last.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        return DeviceArray.from_numpy(np.array([rng.choice(p.shape[-1], p=row) for row in p], np.int32), "int32")
    return pick


def cache_for(num_layers, num_heads, head_dim, page_size=16):
    """new_cache for generate(): just the pages that the requests will need."""
    def make(requests, longest, rows):
        pages = sum(-(-n // page_size) for n in rows)
        return PagedKVCache(pages, page_size, num_heads, head_dim, num_layers, requests, longest)
    return make
