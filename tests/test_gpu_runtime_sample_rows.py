"""Runtime.sample where the last call left no output rows: nothing to draw from, so it is refused, as predictions()
is empty."""
import pytest

import plamo_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def runtime(model_dir):
    rt = plamo_hip.Runtime(model_dir[0], 96)
    with pytest.raises(plamo_hip.PlamoError) as e:  # before any forward
        rt.sample(0.5)
    assert e.value.code == 1 and rt.predictions() == []
    yield rt
    rt.close()


@pytest.mark.parametrize("tokens", [[2000], [2000, 3000, 4000]])
def test_no_output_rows(runtime, tokens):
    runtime.reset()
    first = runtime.prefill([5000, 6000])
    assert runtime.sample(0.5, top_k=1) == (first, 1.0)
    runtime.forward(tokens, output=False)
    for slot in (0, 1):
        with pytest.raises(plamo_hip.PlamoError) as e:
            runtime.sample(0.5, slot=slot)
        assert e.value.code == 1
    again = runtime.forward([7000])
    assert runtime.sample(0.5, top_k=1) == (again, 1.0)


def test_after_reset(runtime):
    runtime.reset()
    runtime.prefill([5000, 6000])
    runtime.reset()
    with pytest.raises(plamo_hip.PlamoError) as e:
        runtime.sample(0.5)
    assert e.value.code == 1
    ids, _ = runtime.generate([5000, 6000], 2)
    assert runtime.sample(0.5, temperature=0.0)[0] == runtime.predictions()[0] and ids
