"""Runtime.sample: tokens drawn from the runtime's own logits, against a 64-bit implementation on the logits
that it hands out."""
import math

import numpy as np
import pytest

import plamo_hip
from paged_common import sample64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def runtime(model_dir):
    rt = plamo_hip.Runtime(model_dir[0], 96)
    yield rt
    rt.close()


def test_a_sampled_loop(runtime):
    runtime.reset()
    rng = np.random.default_rng(21)
    runtime.prefill([1024 + 37 * i for i in range(20)])
    for step in range(12):
        own = {"temperature": float(np.float32(rng.uniform(0.5, 1.5))), "top_k": int(rng.integers(0, 60)),
               "top_p": float(np.float32(rng.uniform(0.5, 1.2))), "min_p": float(np.float32(rng.choice([0.0, 0.02])))}
        u = float(rng.random(dtype=np.float32))
        before = runtime.position, runtime.predictions(), runtime.logit_bits()
        token, prob = runtime.sample(u, **own)
        want, share = sample64(runtime.logits().astype(np.float64), u, **own)
        assert token == want and abs(prob - share) <= 2.0 ** -23 * share + 1e-12, (step, own)
        after = runtime.position, runtime.predictions(), runtime.logit_bits()
        assert before[:2] == after[:2] and np.array_equal(before[2], after[2])
        runtime.forward([token])


def test_greedy_is_the_prediction(runtime):
    runtime.reset()
    first = runtime.prefill([2000, 3000, 4000])
    assert runtime.sample(0.9, temperature=0.0) == (first, 1.0)
    assert runtime.sample(0.9, top_k=1) == (first, 1.0)


@pytest.mark.parametrize("changed", [dict(uniform=1.0), dict(uniform=-0.1), dict(uniform=math.nan), dict(slot=1), dict(slot=-1),
                                     dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=math.nan),
                                     dict(min_p=math.nan)])
def test_refused(runtime, changed):
    runtime.reset()
    runtime.prefill([2000, 3000, 4000])
    call = dict(uniform=0.5)
    call.update(changed)
    with pytest.raises(plamo_hip.PlamoError) as e:
        runtime.sample(**call)
    assert e.value.code == 1
