"""What paged_append stores in an 8-bit cache is the value divided by the scale."""
import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quotients_between_two_values(dtype):
    """Quotients as near the middle of two e4m3 values as fp32 scales allow, at position 0 (nothing is turned): the quotient in fp32,
    rounded once, for k and v."""
    heads, dim = 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    values = torch.arange(1, 126, device="cuda", dtype=torch.uint8).view(E4M3).float()
    middle = ((values[1:] + values[:-1]) / 2)[torch.randint(0, 124, (heads,), device="cuda", generator=g)]
    first = torch.randn(heads, device="cuda", generator=g).to(dtype).float()
    x = (first.abs() + 2.0 ** -10)[:, None].to(dtype) * torch.tensor([1.0, -1.0], device="cuda", dtype=dtype).repeat(dim // 2)
    scale = x[:, 0].float() / middle  # (so the quotient is the middle to half a step of fp32)
    for sc in (scale, torch.nextafter(scale, scale * 2), torch.nextafter(scale, scale * 0)):
        k, v = (torch.zeros(1, 1, heads, dim, device="cuda").to(E4M3) for _ in range(2))
        P.paged_append(torch.cat([x.flatten()] * 2)[None], k, v, torch.zeros(1, dtype=torch.int64, device="cuda"),
                       torch.zeros(1, dtype=torch.int32, device="cuda"), 0, 1e4, k_scale=sc, v_scale=sc)
        want = (x.float() / sc[:, None]).clamp(-448, 448).to(E4M3).float()
        assert torch.equal(k[0, 0].float(), want) and torch.equal(v[0, 0].float(), want)


def test_scales_that_have_no_reciprocal():
    """A scale so small that one over it is no number of fp32: zeros stay zeros, small values keep theirs, others are at the ends."""
    k, v = (torch.full((1, 1, 1, 64), 9.0, device="cuda").to(E4M3) for _ in range(2))
    x = torch.zeros(1, 128, device="cuda", dtype=torch.bfloat16)
    x[0, 65], x[0, 66], x[0, 67] = 2.0 ** -126, -1.0, 2.0 ** -133
    scale = torch.full((1,), 2.0 ** -130, device="cuda")
    P.paged_append(x, k, v, torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 0, 1e4, k_scale=scale,
                   v_scale=scale)
    assert (k.float() == 0).all() and v[0, 0, 0, :5].tolist() == [0, 16, -448, 0.125, 0] and (v[0, 0, 0, 4:].float() == 0).all()
