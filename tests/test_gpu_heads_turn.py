"""Cosines and sines of the rotation in fp32."""
import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("far", [0, 2000000])
def test_of_angles(far, pairs):
    """Heads of ones and zeros come out as cosines and sines.  An angle within an eighth of a turn rounds to 32 bits once,
    by at most u / 2, the result's last sum by u / 2, and the products inside it, which are smaller than a third of it, by
    another u / 2 with what the series leaves; 64-bit angles are off by 3 * 2^-53 of themselves on either side."""
    from hoard_amd import attn
    m, rot = 4096, 64
    g = torch.Generator().manual_seed(1)
    pos = (torch.randint(0, 5000, (m,), generator=g) + far).to(torch.int32).cuda()
    rope = attn.Rope(pos, attn.rope_freq(rot, 10000.0), None, pairs)
    x = torch.zeros((m, 1, rot), device="cuda")
    if pairs:
        x[..., 0::2] = 1.0
    else:
        x[..., :rot // 2] = 1.0
    got = A.t64(attn.heads_forward(x, rope=rope).q_out)
    angle = A.t64(pos).view(-1, 1, 1) * A.t64(rope.freq)
    c, s = (got[..., 0::2], got[..., 1::2]) if pairs else (got[..., :rot // 2], got[..., rot // 2:])
    bound = 1.5 * A.U32 + 6 * 2.0 ** -53 * angle.abs()
    for name, y, want in (("cos", c, torch.cos(angle)), ("sin", s, torch.sin(angle))):
        A.close(y, want, bound, name)
