"""copy_kv_blocks (HIP) against indexing, bit for bit."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("shape,dtype", [((2, 3, 40, 16, 2, 64), torch.bfloat16), ((40, 16, 1, 64), torch.bfloat16),
                                         ((2, 2, 40, 256, 4, 64), torch.bfloat16), ((1, 40, 3, 1, 16), torch.uint8),
                                         ((2, 1, 40, 5, 3, 16), torch.float32), ((2, 12, 40, 48, 8, 128), torch.bfloat16)])
@pytest.mark.parametrize("n", [1, 7, 20])
def test_copies(shape, dtype, n):
    rng = np.random.default_rng(n)
    g = torch.Generator(device=DEV).manual_seed(n)
    pool = torch.randint(0, 250, shape, generator=g, device=DEV).to(dtype)
    ids = rng.permutation(40)
    src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
    want = pool.clone()
    want[..., dst, :, :, :] = pool[..., src, :, :, :]
    K.copy_kv_blocks(pool, src, torch.tensor(dst))
    assert torch.equal(pool, want)


def test_one_block_to_many_and_more_pairs_than_a_launch_takes():
    rng = np.random.default_rng(2)
    pool = torch.randn(2, 2, 2100, 16, 1, 64, device=DEV).to(torch.bfloat16)
    ids = rng.permutation(2100)
    for src, dst in (([int(ids[0])] * 5, ids[1:6].tolist()), (ids[:1000].tolist(), ids[1000:2000].tolist()),
                     (ids[:448].tolist(), ids[448:896].tolist()), (ids[:449].tolist(), ids[449:898].tolist())):
        want = pool.clone()
        want[:, :, dst] = pool[:, :, src]
        K.copy_kv_blocks(pool, src, dst)
        assert torch.equal(pool, want)
    K.copy_kv_blocks(pool, [], [])
    assert torch.equal(pool, want)


def test_pool_past_32_bit_offsets():
    pool = torch.zeros(2, 1, 33000, 256, 4, 64, device=DEV, dtype=torch.bfloat16)
    pool[1, 0, 32999] = 3
    K.copy_kv_blocks(pool, [32999], [32001])
    assert (pool[1, 0, 32001] == 3).all() and (pool[0, 0, 32001] == 0).all() and (pool[1, 0, 32000] == 0).all()


def test_in_a_graph():
    pool = torch.randn(2, 2, 10, 16, 2, 64, device=DEV).to(torch.bfloat16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.copy_kv_blocks(pool, [3, 3], [4, 5])
    for _ in range(3):
        pool.copy_(torch.randn(2, 2, 10, 16, 2, 64, device=DEV))
        want = pool.clone()
        want[:, :, [4, 5]] = pool[:, :, [3, 3]]
        g.replay()
        assert torch.equal(pool, want)


def test_refusals():
    pool = torch.zeros(2, 2, 10, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
    before = pool.clone()
    for src, dst, why in (([0], [10], "outside"), ([-1], [2], "outside"), ([0, 1], [2, 2], "twice"),
                          ([0, 1], [1, 2], "source and a destination"), ([3], [3], "source and a destination"),
                          ([2 ** 40], [0], "outside")):
        with pytest.raises(ValueError, match=why):
            K.copy_kv_blocks(pool, src, dst)
    with pytest.raises(AssertionError, match="same length"):
        K.copy_kv_blocks(pool, [1, 2], [3])
    with pytest.raises(ValueError, match="host data"):
        K.copy_kv_blocks(pool, torch.tensor([1], device=DEV), [3])
    with pytest.raises(ValueError, match="16 bytes"):
        K.copy_kv_blocks(torch.zeros(4, 1, 1, 3, device=DEV), [1], [3])
    with pytest.raises(AssertionError, match="contiguous"):
        K.copy_kv_blocks(pool.transpose(0, 1), [1], [3])
    with pytest.raises(ValueError, match="GPU only"):
        K.copy_kv_blocks(pool.cpu(), [1], [3])
    assert torch.equal(pool, before)
