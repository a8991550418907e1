import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, 'deepgemm-amd_amd')
for p in (ROOT, PKG, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line('markers', 'gpu: needs an MI355X (gfx950) GPU')


@pytest.fixture(autouse=True)
def process_settings():
    """The library's settings (CU count, tile override, MK alignment) back to their defaults
    after every test: set_num_sms has no value for the device's own count, so a test that
    puts back what it read leaves an override behind."""
    yield
    deep_gemm = sys.modules.get('deep_gemm')
    if deep_gemm is not None and hasattr(deep_gemm, 'init'):
        deep_gemm.init()
