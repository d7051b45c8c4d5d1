"""The two in-place forms that the C header promises -- linear's residual in y's own buffer, the activation gradient dz in dy's own buffer -- against the calls with buffers
of their own, bit for bit, for every kernel that a size can reach: kernels that read ahead, and ragged vectors that are read moved back over what a neighbour stores."""
import pytest
import torch

from tests.test_gpu_row_ops import dtype, randn  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu

# few rows; register-staged (ragged K, and shorter than a vector); LDS-DMA tiles with whole and ragged columns, all three of their sizes; 256 x 256 tiles (ragged columns, long K); rows in
# registers, whole and ragged, one to four steps of K, several units a block
SHAPES = [(1, 7, 3), (33, 45, 77), (64, 512, 128), (300, 777, 61), (130, 5, 9), (5001, 1001, 333), (300, 128, 77), (2048, 512, 1024), (5001, 1000, 333), (24600, 128, 520), (9000, 1024, 2048),
          (70001, 120, 320), (131112, 200, 128), (16384, 384, 1024), (16389, 512, 1024), (33333, 333, 520), (70001, 121, 320), (131112, 201, 128), (16389, 505, 1025)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act,pre", [(0, False), (2, True)])
def test_residual_in_the_output_buffer(dtype, m, k, n, act, pre):
    from simhand_amd import _lib, ops

    if dtype == torch.float32:
        m = m // 16 + 5 if m > 10000 else m
    lib, d, st = _lib.load(), ops.dt(dtype), torch.cuda.current_stream().cuda_stream
    x, w, res = (randn(*s, seed=i, scale=0.1, dtype=dtype).cuda() for i, s in enumerate(((m, k), (n, k), (m, n))))
    b = randn(n, seed=5).cuda()
    for shift in (0, 1):  # at a 16-byte address and one element behind it
        buf = torch.empty(m * n + 8, dtype=dtype, device="cuda")
        y = buf[shift:shift + m * n].view(m, n)
        aligned = 1 if (x.data_ptr() | w.data_ptr() | y.data_ptr()) & 15 == 0 else 0
        nb = lib.simhand_linear_fwd_workspace_bytes(m, k, n, d, aligned)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        p = torch.empty(m, n, dtype=dtype, device="cuda") if pre else None
        rbuf = torch.empty_like(buf)
        rr = rbuf[shift:shift + m * n].view(m, n).copy_(res)  # the residual in a buffer of its own, at the same alignment
        outs = []
        for r in (rr, y):
            y.copy_(res)
            assert lib.simhand_linear_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), act, r.data_ptr(), y.data_ptr(), p.data_ptr() if pre else 0, m, k, n, d,
                                          ws.data_ptr() if nb else 0, nb, st) == 0
            outs.append((y.clone(), p.clone() if pre else y))
        assert torch.equal(outs[0][0], outs[1][0]) and (not pre or torch.equal(outs[0][1], outs[1][1])), shift
        assert torch.equal(rr, res)


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 3), (40, 7), (300, 9), (7, 64), (5000, 33), (513, 128), (2050, 77), (64, 2048), (333, 2049), (40000, 100)])
@pytest.mark.parametrize("act", [1, 2, 3])
def test_gradient_in_the_incoming_gradient_buffer(dtype, rows, cols, act):
    from simhand_amd import _lib, ops

    lib, d, st = _lib.load(), ops.dt(dtype), torch.cuda.current_stream().cuda_stream
    dy, z = randn(rows, cols, dtype=dtype).cuda(), (2 * randn(rows, cols, seed=1)).to(dtype).cuda()
    nb = lib.simhand_linear_act_bwd_workspace_bytes(rows, cols, d)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    want, db = torch.empty_like(dy), torch.empty(2, cols, device="cuda")
    assert lib.simhand_linear_act_bwd(dy.data_ptr(), z.data_ptr(), act, want.data_ptr(), db[0].data_ptr(), rows, cols, d, ws.data_ptr() if nb else 0, nb, st) == 0
    for shift in (0, 1):
        buf = torch.empty(rows * cols + 8, dtype=dtype, device="cuda")
        v = buf[shift:shift + rows * cols].view(rows, cols).copy_(dy)
        assert lib.simhand_linear_act_bwd(v.data_ptr(), z.data_ptr(), act, v.data_ptr(), db[1].data_ptr(), rows, cols, d, ws.data_ptr() if nb else 0, nb, st) == 0
        assert torch.equal(v, want) and torch.equal(db[0], db[1]), shift
