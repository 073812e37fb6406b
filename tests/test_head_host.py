"""CPU: what the output head's operators refuse, and the size queries of their C entries."""
import pytest
import torch


def test_cpu_tensors_are_refused():
    from dig_amd import _hip, ops
    x, w, t = torch.randn(4, 64), torch.randn(10, 64), torch.zeros(4, dtype=torch.int64)
    for f in (lambda: ops.layer_norm(x), lambda: ops.linear_cross_entropy(x, w, t),
              lambda: ops.linear_distillation(x, w, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))):
        with pytest.raises(_hip.Dig3dError):
            f()
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t, reduction='avg')


def test_row_norm_partials():
    from dig_amd import _hip
    q = lambda *a: _hip.query('dig3d_rownorm_bwd_blocks', *a)
    assert q(0, 128, 0) == 0 and q(5, 0, 0) == 0 and q(5, 8, 3) == 0
    assert q(1, 128, 0) == 1
    assert q(608, 128, 0) == 76                    # 32 lanes a row, 8 rows a workgroup
    assert q(608, 128, 1) == 38                    # 16 lanes a row
    assert 1 <= q(10 ** 6, 1024, 1) <= 4096
    assert q(5, 1 << 25, 0) == 0 and q(5, (1 << 25) - 1, 0) >= 1


def test_head_workspace():
    from dig_amd import _hip
    q = lambda dt, N, D, V, bwd, needs, ptr=0, ld=None: _hip.query('dig3d_head_ws_kib', dt, ptr, ld or D, ptr, ld or D, N, D, V, bwd, needs)
    for bad in ((3, 4, 64, 10), (0, 0, 64, 10), (0, 4, 0, 10), (0, 4, 64, 0)):
        assert q(*bad, 0, 0) < 0
    assert q(0, 4, 64, 10, 0, 0, ld=63) < 0                                   # a pitch below the width
    assert q(1, 1 << 20, 64, 1 << 27, 0, 0) < 0                               # more tiles than the kernels index
    assert q(1, 1 << 24, 64, 10, 0, 0) < 0 <= q(1, (1 << 24) - 1, 64, 10, 0, 0)
    # a vocabulary of any size that fits one piece is one piece: e's planes alone would differ by 512 MiB otherwise
    assert q(1, 4096, 1024, 65536, 1, 0) - q(1, 4096, 1024, 65535, 1, 0) < 1024
    # 16-bit rows of whole k steps are read in place; odd widths, odd pitches and odd addresses are copied
    direct = q(1, 64, 128, 40960, 0, 0)
    assert direct < q(1, 64, 127, 40960, 0, 0) and direct < q(1, 64, 128, 40960, 0, 0, ptr=2) and direct < q(1, 64, 128, 40960, 0, 0, ld=129)
    assert q(1, 32, 128, 1024, 0, 0) == q(1, 32, 128, 1024, 0, 0, ptr=2)      # small products read anything in place
    # the backward's workspace is bounded in the vocabulary: e in pieces of at most 512 MiB per plane
    big, bigger = q(1, 4096, 1024, 1 << 17, 1, 7), q(1, 4096, 1024, 1 << 20, 1, 7)
    assert bigger <= big + (64 << 10) and bigger < (1 << 21)
