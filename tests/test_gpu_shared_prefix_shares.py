"""Where the kernels over tiles and over rows run side by side they divide the multiprocessors between them by the same count."""
import pytest
import torch

from test_gpu_shared_prefix import PAGE, check, make, run


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 1500, 700])
@pytest.mark.parametrize("hq,hkv,d,warps", [(8, 4, 256, 4), (16, 8, 128, 8)])
def test_their_shares_add_up(hq, hkv, d, warps, window, monkeypatch):
    """The first row of a tile may see further back than the others behind a window, or less far, or nothing of what they share."""
    from kapel_b200 import kernels as K

    if not K.PDL:
        pytest.skip("launches are not chained: one kernel after the other")
    scratch, fresh = [], K._fresh

    def watched(shape, dtype, device):
        t = fresh(shape, dtype, device)
        if len(shape) == 1 and dtype == torch.float32:
            scratch.append(t)
        return t

    monkeypatch.setattr(K, "_fresh", watched)
    blocks = torch.cuda.get_device_properties(0).multi_processor_count
    for counts in ([2400 + 7 * i for i in range(1, 41)], [2400 + 7 * i for i in range(40, 0, -1)], [4000] + [2401 + 50 * i for i in range(30)], [2401] + [3300] * 30):
        scratch.clear()
        c = make([(counts, 2400), ([2900 + i for i in range(6)], 2000)], hq, hkv, d, extra_width=-(-150_000_000 // (len(counts) * PAGE * hkv * d * 4)))
        check(c, window=window, softcap=50.0)
        tiles, tile_workers, row_workers = scratch[-1].view(torch.int32)[-3:].tolist()
        assert tiles > 0 and tile_workers > 0 and row_workers > 0
        assert tile_workers + -(-row_workers // warps) == blocks, (counts[0], tile_workers, row_workers)
