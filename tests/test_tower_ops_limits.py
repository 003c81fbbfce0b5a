"""The encoder towers' operators on the CPU: sizes that their kernels' counters do not hold are refused before anything is launched."""
import torch

EINVAL, EALIGN, ELIMIT = -1, -2, -3


def test_gn_entries_refuse_maps_beyond_their_row_counters():
    """A sample's positions are counted in 32 bits: 2^30 of them are taken, one more is refused, forward and backward."""
    from creamfl_amd import _lib
    lib = _lib.load()
    P, most = 4096, 1 << 30
    assert lib.cfl_gn_ws_bytes(1, most, 8, 1) > 0
    for hw in (most + 1, (1 << 31) - 1):
        assert lib.cfl_gn_ws_bytes(1, hw, 8, 1) == 0
        assert lib.cfl_gn_fwd(P, None, P, P, 1, 1, hw, 8, 1, 1e-5, 0, P, P, P, P, None) == ELIMIT
        assert lib.cfl_gn_bwd(P, None, P, None, P, P, P, P, 1, 1, hw, 8, 1, 0, 0, P, None, P, P, P, None) == ELIMIT


def test_gn_act_refuses_maps_beyond_its_row_counters():
    """[1, 8, 65536, 65537] bf16 fits the card's memory; its positions would reach the entry modulo 2^32 (as 65536)."""
    import pytest
    from torch._subclasses.fake_tensor import FakeTensorMode
    from creamfl_amd import _lib, ops
    with FakeTensorMode():
        def fmap(h, w):
            return torch.empty_strided((1, 8, h, w), (8 * h * w, 1, 8 * w, 8), dtype=torch.bfloat16, device='cuda')
        assert ops.gn_act_supported(fmap(1 << 15, 1 << 15), 8, 1)
        for h, w in ((1 << 15, (1 << 15) + 1), (46340, 46341), (65536, 65537), (1, (1 << 30) + 1)):
            x = fmap(h, w)
            assert not ops.gn_act_supported(x, 8, 1), (h, w)
            with pytest.raises(_lib.CreamflHipError, match='H W'):
                ops.gn_act(x, x, x, 1)
