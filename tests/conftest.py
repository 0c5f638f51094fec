"""pytest configuration: `gpu` marker = needs a real MI355X (run with -m gpu on the GPU box)."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"), os.path.join(ROOT, "ggml-gfx906_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: test needs an MI355X (gfx950) GPU")
    config.addinivalue_line("markers", "slow: long-running test")


def pytest_collection_modifyitems(items):
    """where the reference's programs are not built (oracle/_ref), the tests that want them without asking come last, so
    that a run that ends at its first failure has run all others"""
    if not os.path.exists(os.path.join(ROOT, "oracle", "_ref", "gpt2_ref")):
        items.sort(key=lambda item: item.name in WANT_REFERENCE)


WANT_REFERENCE = {"test_bench_two_ranks_one_gpu_rehearsal"}   # (its line has a leg of the reference's scheduler)
