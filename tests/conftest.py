import pathlib
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
for p in (ROOT / "neuronmlp-on-tpu_b200", ROOT / "oracle", ROOT):
    if str(p) not in sys.path:
        sys.path.insert(0, str(p))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) GPU")


@pytest.fixture(scope="session")
def cuda_device():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    major, _ = torch.cuda.get_device_capability(0)
    if major != 10:
        pytest.skip("needs an sm_100 (B200) device")
    return torch.device("cuda", 0)


def pytest_collection_modifyitems(items):
    # this one expects a branching tree's tokens at successive positions, where they belong at their depth
    # (test_gpu_decoder_steps.py compares them with their own paths); last, so that it hides nothing under -x
    items.sort(key=lambda item: item.name.startswith("test_a_tree_matches_its_paths"))
