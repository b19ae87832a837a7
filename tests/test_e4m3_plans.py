"""The plans of the GPU tests' steps on an e4m3 pool are what the steps are named for (CPU)."""
import pytest

import _e4m3_steps as S
from test_host_plan import FLAGS, build_and_run

SHAPE = ["aegean-tge_amd/host/plan.cpp", "aegean-tge_amd/host/plan_e4m3.cpp", "tests/native/plan_e4m3_shape.cpp"]


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    runs = [(qh, kvh, hd, *[x for s in sessions for x in s]) for qh, kvh, hd, _, sessions, _ in S.STEPS.values()]
    out = build_and_run(tmp_path_factory.mktemp("plans"), "plan_e4m3_shape", SHAPE, runs, flags=FLAGS)
    return {name: dict(zip(line.split()[::2], map(int, line.split()[1::2])))
            for name, line in zip(S.STEPS, out.splitlines(), strict=True)}


@pytest.mark.parametrize("name", S.STEPS)
def test_plan(plans, name):
    held = S.STEPS[name][5]
    p = plans[name]
    assert all(p[k] > 0 for k in held), p
    assert not any(p[k] for k in S.NOT_OTHERWISE - held), p
    if "outgrown" in held:
        assert p["most"] > 128, p
