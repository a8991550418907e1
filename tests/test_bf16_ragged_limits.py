"""Launches of 2^32 threads or more of the ragged BF16 products are refused by the plan, which
the workspace query and the calls share: before any kernel of the call is queued."""
import pytest
import torch

import deep_gemm
from deep_gemm import _ffi

NT, NN, TN, TN8 = 0, 1, 2, 3


@pytest.fixture
def cus():
    deep_gemm.set_num_sms(256)
    yield
    deep_gemm.init()


def size(form, rows, m, n, k, groups, block=0, pieces=0):
    if block:
        deep_gemm.set_tile_override(block, pieces, variant=13)
    got = _ffi.lib.dg_bf16_gemm_ragged_workspace_size(form, rows, m, n, k, groups)
    assert got >= 0 or '<< 32' in _ffi.lib.dg_last_error().decode()
    deep_gemm.set_tile_override(0, 0)
    return got


@pytest.mark.parametrize('form', [NT, NN])
@pytest.mark.parametrize('block', [32, 128, 256])
def test_rows_of_tiles(cus, form, block):
    """One group: rows / tile + 1 row blocks, 8 or 4 column blocks; 2^24 workgroups of 256
    threads or 2^23 of 512 are one too many."""
    most = (1 << 21) - 2            # (most + 1) x 8 x 256 or (most + 1) x 4 x 512 threads
    assert size(form, most * block, 0, 1024, 8, 1, block, block < 256) == 0
    assert size(form, (most + 1) * block, 0, 1024, 8, 1, block, block < 256) == -1


@pytest.mark.parametrize('form', [NT, NN, TN, TN8])
def test_heuristic(cus, form):
    assert size(form, 1 << 29, 1 << 20, 1 << 22, 1 << 20, 65536) == -1
    assert size(form, 1 << 20, 4096, 4096, 4096, 1024) == 0


@pytest.mark.parametrize('form', [TN, TN8])
def test_tiles_of_outputs(cus, form):
    """65536 groups: 248 tiles each of 128 x 128 launch, 256 do not."""
    assert size(form, 100, 1, 248 * 128, 0, 65536, 128, 1) == 0
    assert size(form, 100, 1, 249 * 128, 0, 65536, 128, 1) == -1
    assert size(form, 100, 1, 120 * 256, 0, 65536, 256) == 0
    assert size(form, 100, 1, 121 * 256, 0, 65536, 256) == -1


def test_pieces_sums(cus):
    """The kernel that adds the pieces has a workgroup for every 1024 columns of a row."""
    assert size(NT, (1 << 24) - 1, 0, 8, 8, 1, 128, 2) == ((1 << 24) - 1) * 8 * 4 * 2
    assert size(NT, 1 << 24, 0, 8, 8, 1, 128, 2) == -1


@pytest.mark.gpu
def test_refused_call_writes_nothing():
    dev = 'cuda:0'
    d = torch.full((65536, 1, 256 * 128), 7.0, dtype=torch.bfloat16, device=dev)
    a, b = torch.ones((1, 1), dtype=torch.bfloat16, device=dev), torch.ones((1, 256 * 128), dtype=torch.bfloat16, device=dev)
    ends = torch.ones(65536, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match='<< 32'):
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d, ends)
    assert bool((d == 7.0).all())
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d[:8], ends[:8])
    assert bool((d[0] == 1.0).all()) and bool((d[1:8] == 0.0).all()) and bool((d[8:] == 7.0).all())
