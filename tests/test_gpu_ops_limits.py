"""Row counts near 2^31, as far as one GPU's memory holds their arrays."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16 = torch.float16


def test_q4_ids_of_two_billion_rows():
    """The rows behind 2^31 - 65536, where a step to a workgroup's next row leaves 32 bits."""
    from hoard_amd.ops import Q4Weight, q4_matmul
    n = 2**31 - 5
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (3, 1, 16), generator=g, dtype=torch.uint8).cuda()
    w = Q4Weight(codes, torch.full((3, 1, 1), 0.01, dtype=F16, device="cuda"))
    x = torch.randn((1, 32), generator=g).to(F16).cuda()
    three = q4_matmul(x, w, ids=torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")).view(3)
    ids = torch.empty((1, n), dtype=torch.int32, device="cuda")
    step = 1 << 28
    for a in range(0, n, step):
        ids[0, a:a + step] = torch.arange(a, min(n, a + step), device="cuda") % 3
    print("ids made", flush=True)
    y = q4_matmul(x, w, ids=ids)
    torch.cuda.synchronize()
    print("rows done", flush=True)
    for a in range(0, n, step):
        assert torch.equal(y[a:a + step, 0], three[ids[0, a:a + step].long()]), a
