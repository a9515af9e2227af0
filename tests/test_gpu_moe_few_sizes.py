"""The MoE layer for a few tokens where its kernels end and the grouped path begins, and against its formula in fp32."""
import pytest
import torch

from test_gpu_moe_few import composed, inputs, make_stack

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a B200")]

DEV = "cuda"


@pytest.mark.parametrize("E,k,H,I,dtype", [(4, 2, 128, 14336, torch.float16), (16, 8, 144, 1536, torch.bfloat16),
                                           (9, 8, 64, 2048, torch.float16), (3, 1, 8192, 4096, torch.bfloat16),
                                           (32, 32, 512, 256, torch.float16)])
def test_every_number_of_tokens(E, k, H, I, dtype):
    """1 to 17 tokens of layers whose rows fill the shared memory on the way: each the separate calls, bit for bit."""
    import fni8
    from fni8 import moe

    stack = make_stack(E, H, I, E + k)
    for T in range(1, 18):
        x, logits = inputs(T, E, H, dtype, 31 * T)
        topi, topw = moe.route(logits, k, weight_dtype=dtype)
        want = composed(x, topi, topw, stack, "silu")
        assert torch.equal(moe.layer(x, logits, stack, k), want), T
        assert torch.equal(moe.experts(x, topi, topw, stack), want), T
    assert fni8.device_status() == 0


def int8_rows(v):
    """The quantiser's definition: both quotients rounded once. (Tensor by tensor: torch makes a reciprocal and a
    product of a quotient with a plain number, which is another number in one of a few rows.)"""
    top = v.abs().amax(-1, keepdim=True)
    f = torch.full_like(top, 127)
    inv = torch.where(top > 0, f / top, torch.zeros_like(top))
    return torch.round(v * inv).clamp(-127, 127), top / f


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 7, 16])
def test_formula_in_fp32(T, dtype):
    """Elementary torch operations with every rounding of the definition give the layer's values bit for bit: the
    integer sums are below 2^24, so fp32 products hold them, and SiLU is one exp and one quotient on both sides."""
    from fni8 import moe

    E, k, H, I = 32, 8, 512, 384
    stack = make_stack(E, H, I, 3)
    for seed in range(3):
        x, logits = inputs(T, E, H, dtype, 100 * seed + T)
        topi, topw = moe.route(logits, k, weight_dtype=dtype)
        at = topi.reshape(-1).long()
        q, a = (t.repeat_interleave(k, 0) for t in int8_rows(x.float()))
        gu = torch.bmm(stack.w_gu[at].float(), q.unsqueeze(-1)).squeeze(-1)
        assert float(gu.abs().max()) < 2 ** 24
        gate, up = (gu * a * stack.s_gu[at]).to(dtype).float().chunk(2, -1)
        act = (gate / (1 + torch.exp(-gate))).to(dtype).float()
        hq, b = int8_rows((act * up).to(dtype).float())
        y = torch.bmm(stack.w_dn[at].float(), hq.unsqueeze(-1)).squeeze(-1)
        y = (y * b * stack.s_dn[at]).to(dtype).float().view(T, k, H)
        out = torch.zeros(T, H, device=DEV)
        for j in range(k):
            out = out + topw[:, j:j + 1] * y[:, j]
        assert torch.equal(moe.layer(x, logits, stack, k), out.to(dtype))


@pytest.mark.parametrize("T", [1, 4, 16, 40])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_rows_at_any_address(T, offset):
    """x as a view into a flat buffer at an odd place: the values of its copy."""
    from fni8 import moe

    E, k, H, I = 8, 2, 128, 64
    stack = make_stack(E, H, I, 2)
    x, logits = inputs(T, E, H, torch.bfloat16, T)
    flat = torch.empty(offset + T * H, dtype=x.dtype, device=DEV)
    flat[offset:] = x.reshape(-1)
    view = flat[offset:].view(T, H)
    assert view.data_ptr() % 16
    topi, topw = moe.route(logits, k, weight_dtype=x.dtype)
    assert torch.equal(moe.layer(view, logits, stack, k), moe.layer(x, logits, stack, k))
    assert torch.equal(moe.experts(view, topi, topw, stack), moe.experts(x, topi, topw, stack))
