"""The few-token MoE layer: bit for bit the separate calls (route, plan, quantise, grouped GEMMs, combine), and within
a counted bound of the layer's formula in 64 bits."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a B200")]

DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make_stack(E, H, I, seed):
    from fni8.moe import ExpertStack

    g = gen(seed)

    def w(n, k):
        return (torch.randint(-127, 128, (E, n, k), generator=g, device=DEV, dtype=torch.int8),
                (0.5 + torch.rand(E, n, generator=g, device=DEV)) * (2.0 / (127 * k ** 0.5)))

    (gu, sgu), (dn, sdn) = w(2 * I, H), w(H, I)
    return ExpertStack(gu, sgu, dn, sdn)


def composed(x, topi, topw, stack, act):
    """The routed experts from the package's separate calls."""
    import fni8
    from fni8 import moe

    T, k = topi.shape
    E, I = stack.num_experts, stack.intermediate
    counts, offsets, ros, _ = moe.plan(topi, E)
    aq, a_s = moe.quantize_scatter(x, ros, k, T * k)
    seg = torch.arange(E, device=DEV, dtype=torch.int32)
    gu = moe.grouped_gemm(aq, a_s, stack.w_gu, stack.s_gu, seg, offsets[:-1], counts, out_dtype=x.dtype)
    rows = int(offsets[-1])  # rows behind the last expert's are unwritten
    hq = torch.zeros(T * k, I, dtype=torch.int8, device=DEV)
    hs = torch.zeros(T * k, dtype=torch.float32, device=DEV)
    if rows:
        hq[:rows], hs[:rows] = fni8.act_and_mul_quant(gu[:rows], act)
    y = moe.grouped_gemm(hq, hs, stack.w_dn, stack.s_dn, seg, offsets[:-1], counts, out_dtype=x.dtype)
    return moe.combine(y, ros, topw)


def inputs(T, E, H, dtype, seed):
    g = gen(seed)
    x = torch.randn(T, H, generator=g, device=DEV)
    x[:, torch.rand(H, generator=g, device=DEV) < 0.01] *= 20
    return x.to(dtype), 2 * torch.randn(T, E, generator=g, device=DEV)


CASES = [  # T, E, k, H, I, dtype, act
    (1, 128, 8, 2048, 768, torch.float16, "silu"), (16, 128, 8, 2048, 768, torch.bfloat16, "silu"),
    (3, 8, 2, 4096, 1024, torch.float16, "gelu_tanh"), (1, 1, 1, 16, 16, torch.float16, "silu"),
    (16, 1, 1, 48, 32, torch.bfloat16, "gelu_tanh"), (9, 2, 2, 1040, 208, torch.float16, "silu"),
    (5, 33, 7, 272, 400, torch.bfloat16, "silu"), (16, 512, 32, 64, 16, torch.float16, "silu"),
    (2, 300, 4, 144, 2064, torch.float16, "gelu_tanh"), (13, 65, 3, 7168, 128, torch.bfloat16, "silu"),
    (12, 5, 5, 640, 96, torch.float16, "silu"), (7, 64, 6, 1040, 208, torch.float16, "gelu_tanh"),
]


@pytest.mark.parametrize("T,E,k,H,I,dtype,act", CASES)
def test_layer_is_the_separate_calls(T, E, k, H, I, dtype, act):
    import fni8
    from fni8 import moe

    stack = make_stack(E, H, I, T + E)
    x, logits = inputs(T, E, H, dtype, 7 * T + k)
    topi, topw = moe.route(logits, k, weight_dtype=dtype)
    want = composed(x, topi, topw, stack, act)
    assert torch.isfinite(want).all() and float(want.abs().max()) > 0
    for _ in range(3):
        assert torch.equal(moe.layer(x, logits, stack, k, act=act), want)
        assert torch.equal(moe.experts(x, topi, topw, stack, act), want)
    assert fni8.device_status() == 0


@pytest.mark.parametrize("T", [1, 6, 16, 17, 40])
@pytest.mark.parametrize("norm,scaling,groups", [(True, 1.0, None), (False, 2.5, (8, 3)), (True, 0.7, (4, 1))])
def test_sigmoid_and_grouped_routing(T, norm, scaling, groups):
    from fni8 import moe

    E, k, H, I = 64, 6, 256, 128
    stack = make_stack(E, H, I, T)
    x, logits = inputs(T, E, H, torch.float16, T)
    bias = 0.3 * torch.randn(E, generator=gen(3), device=DEV)
    ng, tg = groups or (None, None)
    for scoring, b in (("sigmoid", bias), ("sigmoid", None), ("softmax", None)):
        topi, topw = moe.route(logits, k, scoring=scoring, sel_bias=b, num_expert_groups=ng, topk_group=tg,
                               norm_topk_prob=norm, scaling=scaling, weight_dtype=x.dtype)
        got = moe.layer(x, logits, stack, k, scoring=scoring, sel_bias=b, num_expert_groups=ng, topk_group=tg,
                        norm_topk_prob=norm, scaling=scaling)
        assert torch.equal(got, composed(x, topi, topw, stack, "silu"))


@pytest.mark.parametrize("T,k", [(1, 8), (4, 32), (16, 32), (16, 3)])
def test_repeated_and_unknown_experts(T, k):
    """Ids given by the caller: the same expert many times over, all tokens to one expert, ids outside [0, E)."""
    from fni8 import moe

    E, H, I = 9, 128, 64
    stack = make_stack(E, H, I, 5)
    x, _ = inputs(T, E, H, torch.float16, 1)
    g = gen(2)
    topw = torch.rand(T, k, generator=g, device=DEV)
    for topi in (torch.full((T, k), 4), torch.randint(0, E, (T, k)), torch.randint(-2, E + 2, (T, k)),
                 torch.full((T, k), -1), torch.full((T, k), 2 ** 31 - 1)):
        ti = topi.to(DEV, torch.int32)
        want = composed(x, ti, topw, stack, "silu")
        assert torch.equal(moe.experts(x, ti, topw, stack), want)
        if int(topi.min()) in (-1, 2 ** 31 - 1) and int(topi.max()) == int(topi.min()):
            assert not want.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_special_values(dtype):
    """Zero rows, infinities and NaN in x, logits that are equal, infinite or NaN: as the separate calls."""
    from fni8 import moe

    T, E, k, H, I = 8, 16, 4, 256, 64
    stack = make_stack(E, H, I, 6)
    x, logits = inputs(T, E, H, dtype, 9)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = torch.finfo(dtype).max
    logits[3] = 0
    logits[4, 2:] = float("-inf")
    logits[5, 7] = float("inf")
    logits[6] = float("nan")
    topi, topw = moe.route(logits, k, weight_dtype=dtype)
    want, got = composed(x, topi, topw, stack, "silu"), moe.layer(x, logits, stack, k)
    assert torch.equal(torch.isnan(want), torch.isnan(got))
    assert torch.equal(torch.nan_to_num(want, nan=7.0), torch.nan_to_num(got, nan=7.0))
    assert not got[0].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 4, 2, 64, 32), (16, 12, 5, 144, 48), (6, 3, 3, 512, 256)])
def test_against_the_formula_in_64_bits(dtype, T, E, k, H, I):
    """x holds whole codes (its rows' largest is 127 times a power of two), the weights' scales are powers of two and
    the gates are large (SiLU(g) = g to the last bit of either type), so everything up to the product act(g) u is
    exact before its rounding. Counted from there: y is off by its rounding (eps / 2) and two fp32 roundings, the
    router's weights by one step of the type, the sum by k + 1 fp32 roundings, the result by its own rounding."""
    from fni8 import moe
    from fni8.moe import ExpertStack

    g = gen(T)
    x = torch.randint(1, 100, (T, H), generator=g, device=DEV).double()
    x[:, 5] = 127
    x = x * torch.exp2(torch.randint(-1, 2, (T, 1), generator=g, device=DEV).double())
    w_gu = torch.randint(-100, 101, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.int8)
    w_gu[:, :I] = w_gu[:, :I].abs() + 1
    w_dn = torch.randint(-127, 128, (E, H, I), generator=g, device=DEV, dtype=torch.int8)
    s_gu = torch.empty(E, 2 * I, device=DEV)  # gates of some hundreds, up values of a few
    s_gu[:, :I] = 2.0 ** -(round(math.log2(2500 * H)) - 9)
    s_gu[:, I:] = 2.0 ** -round(math.log2(3300 * H ** 0.5))
    s_gu *= torch.exp2(torch.randint(-1, 1, (E, 2 * I), generator=g, device=DEV).float())
    s_dn = torch.exp2(torch.randint(-14, -11, (E, H), generator=g, device=DEV).float())
    logits = torch.randn(T, E, generator=g, device=DEV)
    got = moe.layer(x.to(dtype), logits, ExpertStack(w_gu, s_gu, w_dn, s_dn), k).double()

    assert torch.equal(x.to(dtype).double(), x)
    scale = x.abs().amax(-1) / 127
    q = x / scale.unsqueeze(-1)
    w, topi = torch.topk(torch.softmax(logits.double(), -1), k, -1)
    w = w / w.sum(-1, keepdim=True)
    eps = torch.finfo(dtype).eps
    want, tol = torch.zeros(T, H, dtype=torch.float64, device=DEV), torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for t in range(T):
        for j in range(k):
            e = int(topi[t, j])
            gu = ((w_gu[e].double() @ q[t]) * scale[t] * s_gu[e].double()).to(dtype).double()
            assert gu[:I].min() > 40
            h = (gu[:I] * gu[I:]).to(dtype)
            assert torch.isfinite(h).all()
            top = h.float().abs().max()
            codes = torch.round(h.float() * (127.0 / top)).double()  # the quantiser's own fp32 definition
            y = (w_dn[e].double() @ codes) * (top.double() / 127) * s_dn[e].double()
            want[t] += w[t, j] * y
            # y's rounding and denormals, the weight's, the fp32 steps
            tol[t] += w[t, j] * (y.abs() * (eps / 2 + eps + (3 + k + 1) * 2.0 ** -23) + 2.0 ** -25)
    tol = tol + eps / 2 * (want.abs() + tol) + 2.0 ** -25
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def test_graphs_streams_and_views():
    from fni8 import moe

    T, E, k, H, I = 4, 32, 4, 512, 256
    stack = make_stack(E, H, I, 1)
    x, logits = inputs(T, E, H, torch.float16, 1)
    graphs, outs = [], []
    moe.layer(x, logits, stack, k)
    torch.cuda.synchronize()
    for _ in range(2):  # two graphs over the same inputs, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(moe.layer(x, logits, stack, k))
        graphs.append(g)
    for seed in (2, 3):
        nx, nl = inputs(T, E, H, torch.float16, seed)
        x.copy_(nx)
        logits.copy_(nl)
        want = moe.layer(x, logits, stack, k)
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    wide = torch.randn(T, 2 * H, generator=gen(4), device=DEV).half()
    assert torch.equal(moe.layer(wide[:, H:], logits, stack, k), moe.layer(wide[:, H:].contiguous(), logits, stack, k))
    lg = torch.randn(E, T, generator=gen(5), device=DEV).t()
    assert torch.equal(moe.layer(x, lg, stack, k), moe.layer(x, lg.contiguous(), stack, k))
    assert torch.equal(moe.layer(x, logits.half(), stack, k), moe.layer(x, logits.half().float(), stack, k))


@pytest.mark.parametrize("shared", ["none", "int8", "mxfp4", "nvfp4"])
def test_sparse_moe_module(shared):
    """SparseMoE.forward as a model runs it, at decode and prefill sizes, over a shared expert of any scheme."""
    import fni8
    from fni8 import moe
    from fni8.quant.core import quantize_int8_rowwise

    E, k, H, I = 8, 2, 128, 64
    g = torch.Generator().manual_seed(1)

    def qt(n, kk, scheme="int8"):
        w = 0.1 * torch.randn(n, kk, generator=g)
        if scheme == "int8":
            q, s = quantize_int8_rowwise(w)
            return fni8.QTensor(q.to(DEV), s.squeeze(-1).to(DEV))
        return fni8.quantize_fp4(w.half().to(DEV), scheme)

    experts = [(qt(2 * I, H), qt(H, I)) for _ in range(E)]
    sh = None if shared == "none" else (qt(2 * I, H, shared), qt(H, I, shared))
    gate = torch.randn(E, H, generator=g).to(DEV)
    block = moe.SparseMoE(gate=gate, experts=experts, top_k=k, shared_expert=sh)
    for B, S in ((1, 1), (2, 5), (3, 40)):
        x = torch.randn(B, S, H, generator=g).half().to(DEV)
        xf = x.reshape(-1, H)
        topi, topw = moe.route(F.linear(xf.float(), gate.float()), k, weight_dtype=x.dtype)
        want = composed(xf, topi, topw, block.stack, "silu")
        if sh is not None:
            want = want + fni8.linear(fni8.act_and_mul(fni8.linear(xf, sh[0])), sh[1])
        assert torch.equal(block(x), want.reshape(B, S, H))


def test_refusals_on_the_gpu():
    from fni8 import moe

    stack = make_stack(4, 64, 32, 1)
    x, logits = inputs(2, 4, 64, torch.float16, 1)
    for bad in (dict(x=x[:, :48]), dict(logits=logits[:1]), dict(logits=logits[:, :3]), dict(scoring="tanh"),
                dict(act="relu"), dict(sel_bias=torch.zeros(3, device=DEV), scoring="sigmoid")):
        a = {"x": x, "logits": logits, **bad}
        with pytest.raises(ValueError):
            moe.layer(a.pop("x"), a.pop("logits"), stack, 2, **a)
    with pytest.raises(TypeError):
        moe.layer(x.float(), logits, stack, 2)
    for bad_k in (0, 5, 40):
        with pytest.raises(moe.nat.Fni8Error):
            moe.layer(x, logits, stack, bad_k)
    with pytest.raises(moe.nat.Fni8Error):
        moe.layer(x, logits, stack, 2, num_expert_groups=3, topk_group=1)
    with pytest.raises(RuntimeError):
        moe.layer(x, logits.cpu(), stack, 2)
    assert moe.layer(x[:0], logits[:0], stack, 2).shape == (0, 64)
