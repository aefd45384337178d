import gc
import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


def pytest_collection_finish(session):
    """A full garbage collection over what the imports left takes 80 ms, longer than a stream is kept busy by the tests that
    look at what happens meanwhile: those objects are set apart."""
    gc.collect()
    gc.freeze()


@pytest.fixture(scope="module", autouse=True)
def kernels_are_loaded(request):
    """A kernel's first launch loads it, which waits for what the GPU is doing: tests that look at what happens while a
    stream is busy find their kernels loaded, also when they run by themselves, and no garbage is collected meanwhile."""
    if request.module.__name__ != "test_gpu_paged_streams":
        yield
        return
    import torch
    from magpie_tts_rt_b200 import paged_cache as pc
    m = request.module
    cache, groups = m.voices_and_members(pc, [640, 96], [[1, 5, 9], [2, 30, 4]])
    plan = pc.PrefixGroups(cache, groups, q_heads=4)
    plan._c.shared_tokens = 0
    for stream in (None, torch.cuda.Stream()):
        cache.attend_shared(0, m.queries(cache.slots, 4, 64, torch.bfloat16).cuda(), plan, return_lse=True, stream=stream)
        cache.extend(torch.zeros(cache.slots, dtype=torch.int32, device="cuda"), stream=stream)
        torch.cuda._sleep(1)
        torch.cuda.synchronize()
    del cache, plan
    gc.collect()
    gc.disable()
    yield
    gc.enable()


@pytest.fixture(scope="session")
def golden():
    import json
    with open(os.path.join(REPO, "tests", "golden", "golden.json")) as fh:
        return json.load(fh)


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(REPO, "tests", "golden")
