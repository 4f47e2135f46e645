"""The measured cases of perf/operators.py: what they prepare goes when they go."""
import gc
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_dropped_case_gives_its_symmetric_allocation_back(cuda):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    case = {"op": "norm", "T": 64, "H": 1024, "ranks": 4, "dtype": "bf16", "post": True, "gate": "none", "sum": True}
    other = SM.empty_strided_p2p((8,), (1,), torch.bfloat16, cuda, world_size=2, rank=0)
    before = len(SM._by_addr)
    state = cases.prepare(case, 1)
    first = {k: v.clone() for k, v in cases.run(state).items()}
    assert len(SM._by_addr) == before + 4
    second = cases.prepare(case, 2)
    cases.run(second)
    del second
    gc.collect()
    assert len(SM._by_addr) == before + 4
    again = cases.run(state)                                       # the other state's allocation is as it was
    assert all(torch.equal(first[k], again[k]) for k in first)
    del state, again
    gc.collect()
    assert len(SM._by_addr) == before and SM.rendezvous(other) is not None
    SM.release(other)
