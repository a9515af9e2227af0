"""fni8.linear right behind the kernels that write its weight: nothing of it may be read before they have ended."""
import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a B200")]

DEV = "cuda"
SCHEMES = ["mxfp4", "nvfp4"]
# one kernel that quantises x, split-K behind the quantiser (32, 64 and 128 tokens to a block), tiles
ROWS = [1, 16, 17, 64, 128, 300]


def weights(n, N, K, scheme):
    import fni8

    g = torch.Generator(device=DEV).manual_seed(K)
    out = []
    for i in range(n):
        w = fni8.quantize_fp4((0.05 * (i + 1) * torch.randn(N, K, generator=g, device=DEV)).half(), scheme)
        if w.row_scale is not None:
            w.row_scale.mul_(1.0 + 0.37 * i)
        out.append(w)
    return out


def into(dst, src):
    """The weight src into dst's tensors: one small kernel to each part, the row scale last."""
    dst.data.copy_(src.data)
    dst.scale.copy_(src.scale)
    if dst.row_scale is not None:
        dst.row_scale.copy_(src.row_scale)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M", ROWS)
def test_weight_rewritten_in_place(scheme, M):
    import fni8

    N, K = 2304, 4096
    x = torch.randn(M, K, generator=torch.Generator(device=DEV).manual_seed(M), device=DEV).half()
    xq = fni8.quantize_fp4(x, scheme)
    bias = torch.zeros(N, device=DEV).half()
    src = weights(4, N, K, scheme)
    live = weights(1, N, K, scheme)[0]
    want = [fni8.linear(x, w, bias=bias + i) for i, w in enumerate(src)]
    torch.cuda.synchronize()
    got, got_q, order = [], [], [0, 3, 1, 2, 3, 0, 2, 1]
    for i in order:
        into(live, src[i])
        bias.fill_(i)
        got.append(fni8.linear(x, live, bias=bias))
        into(live, src[3 - i])
        bias.fill_(3 - i)
        got_q.append(fni8.linear_fp4(xq, live, bias=bias))
    torch.cuda.synchronize()
    for i, y, yq in zip(order, got, got_q):
        assert torch.equal(y, want[i]) and torch.equal(yq, want[3 - i])
    # only the row scale changes, right in front of the call
    if scheme == "nvfp4":
        ys = []
        for f in (2.0, 0.5, 4.0, 0.25):
            live.row_scale.mul_(f)
            ys.append(fni8.linear(x, live))
        torch.cuda.synchronize()
        for y, f in zip(ys, (1.0, 0.5, 2.0, 0.5)):
            ref = fni8.QTensor(live.data, live.scale, scheme=scheme, row_scale=live.row_scale * (2.0 * f), cols=K)
            torch.cuda.synchronize()
            assert torch.equal(y, fni8.linear(x, ref))
    assert fni8.device_status() == 0


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M", ROWS)
def test_weight_rewritten_within_a_graph(scheme, M):
    import fni8

    N, K = 1152, 2048
    x = torch.randn(M, K, generator=torch.Generator(device=DEV).manual_seed(M), device=DEV).half()
    src = weights(2, N, K, scheme)
    live = weights(1, N, K, scheme)[0]
    want = [fni8.linear(x, w) for w in src]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = []
        for i in (0, 1, 0, 1):
            into(live, src[i])
            ys.append(fni8.linear(x, live))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for y, i in zip(ys, (0, 1, 0, 1)))


@pytest.mark.parametrize("scheme", SCHEMES)
def test_clusters_of_two_streams(scheme):
    """Split-K clusters of every width at once on three streams, short K among them (small CTAs, many to an SM): each
    result is that of the call alone."""
    import fni8

    sizes = [(128, 1536, 4096), (17, 9216, 512), (64, 6144, 768), (16, 12288, 512), (66, 2048, 5120), (20, 4096, 512)]
    g = torch.Generator(device=DEV).manual_seed(1)
    ws = [fni8.quantize_fp4((0.05 * torch.randn(N, K, generator=g, device=DEV)).half(), scheme) for _, N, K in sizes]
    xs = [torch.randn(M, K, generator=g, device=DEV).half() for M, _, K in sizes]
    want = [fni8.linear(x, w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for r in range(40):
        for i in range(len(sizes)):
            with torch.cuda.stream(streams[(i + r) % 3]):
                got.append((i, fni8.linear(xs[i], ws[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    assert fni8.device_status() == 0


@pytest.mark.parametrize("E,k,H,I", [(4, 1, 2048, 16), (16, 4, 512, 256), (64, 6, 1040, 208)])
@pytest.mark.parametrize("T", [1, 3])
def test_routing_and_experts_rewritten_in_place(T, E, k, H, I):
    """The MoE layer directly behind the kernels that write its logits, bias, rows and weights, at the addresses that
    the call before read: layers whose second kernel has more CTAs than the first, eager and in a graph."""
    from fni8 import moe

    g = torch.Generator(device=DEV).manual_seed(T)

    def values():
        def w(n, m):
            return (torch.randint(-127, 128, (E, n, m), generator=g, device=DEV, dtype=torch.int8),
                    (0.5 + torch.rand(E, n, generator=g, device=DEV)) * (2.0 / (127 * m ** 0.5)))

        return (torch.randn(T, H, generator=g, device=DEV).half(), torch.randn(T, E, generator=g, device=DEV),
                0.3 * torch.randn(E, generator=g, device=DEV), *w(2 * I, H), *w(H, I))

    def call(v):
        x, logits, bias, *w = v
        return moe.layer(x, logits, moe.ExpertStack(*w), k, scoring="sigmoid", sel_bias=bias)

    src = [values() for _ in range(4)]
    live = [t.clone() for t in src[0]]
    want = [call(v) for v in src]
    torch.cuda.synchronize()

    def rewrite(v, order):
        for i in order:
            live[i].copy_(v[i])

    got, order = [], [0, 3, 1, 2, 3, 0, 2, 1]
    for n, i in enumerate(order):  # the routing's inputs last, then the weights last
        rewrite(src[i], (0, 3, 4, 5, 6, 2, 1) if n % 2 else (1, 2, 0, 6, 4, 3, 5))
        got.append(call(live))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for y, i in zip(got, order))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = []
        for i in (1, 2, 0):
            rewrite(src[i], (0, 3, 4, 5, 6, 2, 1))
            ys.append(call(live))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for y, i in zip(ys, (1, 2, 0)))
