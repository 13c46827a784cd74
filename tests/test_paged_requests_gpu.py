"""Requests over a paged cache at the edges of what a step may ask for, through both models."""
import numpy as np
import pytest

from tests.test_infer_gpu import cache_of, models
from tests.test_ops_gpu import DTYPES, TOL, close, no_device_flag

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    import mytorch_b200 as m
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,heads,kv_heads", [("gpt2", 2, 2), ("nanochat", 4, 2)])
def test_idle_requests_and_lists_of_other_lengths(mt, dtype, kind, heads, kv_heads):
    """A request without new tokens has zeros, wherever it stands; a list of counts with other zeros at its end asks for as many
    rows as it has counts; the others have the logits of each request alone."""
    model = models(mt, kind, dtype, heads, kv_heads, 64, False)
    r = np.random.default_rng(11)
    ids = [r.integers(0, 200, 30).astype(np.int32) for _ in range(4)]
    cache, alone, at = mt.PagedKVCache(40, 16, kv_heads, 64, 2, 4, 160), [cache_of(mt, model, kind, 1) for _ in ids], [0] * 4
    with mt.no_grad():
        for fresh in ([5, 0, 9], [1, 0, 1], [1, 0, 1, 0], [0, 1, 1, 1], [0, 1, 1, 1], [1, 0], [1], [0, 0, 0, 1]):
            new = [a[i:i + n] for a, i, n in zip(ids, at, fresh)]
            logits = model(mt.Tensor(np.concatenate(new)[None]), cache=cache.begin(fresh))[0].numpy()
            assert logits.shape[:2] == (len(fresh), 1)
            for i, x in enumerate(new):
                at[i] += len(x)
                if len(x):
                    want = model(mt.Tensor(x[None]), cache=alone[i])[0].numpy()[0, -1]
                    close(logits[i, 0], want, 2 * TOL[dtype], f"request {i} of {fresh}")
                else:
                    assert (logits[i] == 0).all(), (i, fresh)
    no_device_flag(mt)


@pytest.mark.parametrize("kind", ["gpt2", "nanochat"])
@pytest.mark.parametrize("lengths,new", [((3, 120, 17), 41), ((160, 9), 1)])
def test_generate_up_to_the_last_position(mt, kind, lengths, new):
    """160 positions: as far as each prompt alone, and no further."""
    model = models(mt, kind, "float32", 2, 2, 64, False)
    r = np.random.default_rng(9)
    prompts = [r.integers(0, 200, n).astype(np.int32) for n in lengths]
    got = model.generate(prompts, new, temperature=0)
    for p, g in zip(prompts, got):
        assert np.array_equal(g, model.generate(p[None], new, temperature=0)[0])
    with pytest.raises(ValueError):
        model.generate(prompts, new + 1, temperature=0)
    no_device_flag(mt)


@pytest.mark.parametrize("kind", ["gpt2", "nanochat"])
def test_a_step_whose_forward_was_refused(mt, kind):
    """Its rows are in no layer: the next step is refused, and after the step was taken back, or run with the right ids, every
    logit is what it is without the refusal."""
    model = models(mt, kind, "float16", 2, 2, 64, False)
    r = np.random.default_rng(5)
    ids = r.integers(0, 200, (3, 60)).astype(np.int32)
    steps = [[20, 7], [1, 16, 30], [1, 1, 1]]

    def run(disturb):
        cache, out, at = mt.PagedKVCache(12, 16, 2, 64, 2, 3, 60), [], [0] * 3
        for n, fresh in enumerate(steps):
            new = np.concatenate([a[i:i + m] for a, i, m in zip(ids, at, fresh)])[None]
            at = [i + (fresh[k] if k < len(fresh) else 0) for k, i in enumerate(at)]
            cache.begin(fresh)
            if disturb:
                with pytest.raises(ValueError):
                    model(mt.Tensor(new[:, :-1]), cache=cache)
                with pytest.raises(RuntimeError):
                    cache.begin(fresh)
                if n != 1:
                    cache.cancel()
                    assert np.array_equal(cache.kv_len.numpy(), cache.lengths)
                    cache.begin([2]).cancel()                    # another step, taken back too
                    cache.begin(fresh)
            out.append(model(mt.Tensor(new), cache=cache)[0].numpy())
            assert np.array_equal(cache.kv_len.numpy(), cache.lengths)
        return out
    with mt.no_grad():
        for a, b in zip(run(True), run(False)):
            assert np.array_equal(a, b)
    no_device_flag(mt)
