"""rms_norm_quant_fp8 against its definition in 64 bits.

Tolerances.  The residual is one addition and one rounding: equal bits.  y: the mean of squares is a tree of fp32 additions (at most 16
in a thread, 5 + 5 in the reductions), whose relative error halves under the root; with the divisions, the root and two products y is
off by at most 24 * 2^-24 of itself.  The norm adds its rounding (2^-8 bf16, 2^-24 fp32), the scale one division, a value at most half
a step of e4m3: 2^-4 of it, or 2^-10 of the scale where it is subnormal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
Y = 24 * 2.0 ** -24


def fg():
    import flaggems_sglang_b200 as m

    return m


def make(rows, K, dtype, seed, residual):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, K, generator=g, device="cuda")
    x[:, :: max(1, K // 3)] *= 30.0
    r = (2 * torch.randn(rows, K, generator=g, device="cuda")).to(dtype) if residual else None
    return x.to(dtype), r, 1 + 0.2 * torch.randn(K, generator=g, device="cuda")


def check(x, weight, eps, residual, per_token, got, residual_after):
    h = x
    if residual is not None:
        h = (x.float() + residual.float()).to(x.dtype)
        assert torch.equal(residual_after, h)
    h = h.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    q, s, norm = got
    g = y.view(y.shape[0], -1, y.shape[1] if per_token else 128)
    amax = g.abs().amax(-1)
    want = (amax / 448).clamp_min(1 / (448 * 512)) if per_token else amax.clamp_min(1e-10) / 448
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    sd = s.double().view(want.shape)
    assert ((sd - want).abs() <= want * (Y + 2.0 ** -23)).all()
    off = ((q.double().view(g.shape) * sd[..., None]) - g).abs()
    assert (off <= g.abs() * (2.0 ** -4 + 2 * Y) + sd[..., None] * (2.0 ** -10 + 448 * Y)).all()
    if norm is not None:
        half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
        assert norm.dtype == x.dtype and ((norm.double() - y).abs() <= y.abs() * (half + 2 * Y) + 1e-38).all()


@pytest.mark.parametrize("rows,K", [(1, 128), (1, 7168), (2, 256), (3, 1152), (17, 4096), (5, 8192), (4, 8320), (2, 16384), (700, 2048), (5000, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("per_token", [False, True])
def test_norm(rows, K, dtype, residual, per_token):
    x, r, w = make(rows, K, dtype, rows + K, residual)
    w = w.to(dtype)
    keep, before = x.clone(), None if r is None else r.clone()
    got = fg().rms_norm_quant_fp8(x, w, 1e-6, residual=r, per_token=per_token, return_norm=True)
    check(x, w, 1e-6, before, per_token, got, r)
    assert torch.equal(x, keep)
    if r is not None:
        r.copy_(before)
    q, s = fg().rms_norm_quant_fp8(x, w, 1e-6, residual=r, per_token=per_token)
    assert torch.equal(q.view(torch.uint8), got[0].view(torch.uint8)) and torch.equal(s, got[1])


@pytest.mark.parametrize("K", [8, 40, 200, 2880, 5672])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_per_token_rows_of_odd_length(K, dtype):
    x, r, w = make(9, K, dtype, K, True)
    before = r.clone()
    got = fg().rms_norm_quant_fp8(x, w, 1e-5, residual=r, per_token=True, return_norm=True)
    check(x, w, 1e-5, before, True, got, r)


def test_bf16_rows_with_fp32_weight_strides_and_itself_as_residual():
    big, _, w = make(6, 1024, torch.bfloat16, 3, False)
    x = big[:, 256:768]
    assert not x.is_contiguous()
    w = w[:512]
    check(x, w, 1e-6, None, False, fg().rms_norm_quant_fp8(x, w, return_norm=True), None)
    store = torch.zeros(6, 1024, dtype=torch.bfloat16, device="cuda")
    r = store[:, 512:]
    r.copy_(big[:, :512])
    before = r.clone()
    check(x, w, 1e-6, before, False, fg().rms_norm_quant_fp8(x, w, residual=r, return_norm=True), r)
    assert (store[:, :512] == 0).all()
    odd = torch.empty(6 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 512)
    odd.copy_(x)
    check(odd, w, 1e-6, None, False, fg().rms_norm_quant_fp8(odd, w, return_norm=True), None)
    same = x.contiguous()
    before = same.clone()
    got = fg().rms_norm_quant_fp8(same, w, residual=same, return_norm=True)
    check(before, w, 1e-6, before, False, got, same)


def test_zeros_infinities_and_no_rows():
    w = torch.ones(256, device="cuda")
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    x[3] = 1
    q, s, n = fg().rms_norm_quant_fp8(x, w, return_norm=True)
    assert (q[0].float() == 0).all() and (n[0] == 0).all()
    assert not torch.isfinite(n[1, 3]) and torch.isnan(n[2]).all()
    check(x[3:], w, 1e-6, None, False, (q[3:], s[3:], n[3:]), None)
    q, s = fg().rms_norm_quant_fp8(x[:0], w)
    assert q.shape == (0, 256) and s.shape == (0, 2)


def test_quantised_output_is_what_the_quantiser_makes_of_the_fp32_norm():
    x, _, w = make(50, 1280, torch.float32, 9, False)
    q, s, n = fg().rms_norm_quant_fp8(x, w, return_norm=True)
    q2, s2 = fg().per_token_group_quant_fp8(n)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


def test_refusals():
    f = fg().rms_norm_quant_fp8
    x, w = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda"), torch.ones(256, device="cuda")
    for bad in (dict(x=x[0]), dict(x=x.half()), dict(weight=w[:128]), dict(weight=w.half()), dict(x=x[:, :200], weight=w[:200]),
                dict(x=torch.zeros(1, 16512, dtype=torch.bfloat16, device="cuda"), weight=torch.ones(16512, device="cuda")),
                dict(residual=x.float()), dict(residual=x[:1]), dict(residual=torch.zeros(256, 2, dtype=torch.bfloat16, device="cuda").t()),
                dict(x=x[:, :4], weight=w[:4], per_token=True)):
        with pytest.raises(ValueError):
            f(**{**dict(x=x, weight=w), **bad})
    with pytest.raises(RuntimeError):
        f(x.cpu(), w)


def test_norm_feeds_the_layer():
    """The run of them as a layer has it: norm -> {router and routed experts, shared expert} -> sum, eager and replayed."""
    m = fg()
    T, H, I, E = 12, 512, 256, 8
    g = torch.Generator(device="cuda")
    g.manual_seed(4)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    w13, s13 = m.quant_weight_block128(rand(E, 2 * I, H) / H ** 0.5)
    w2, s2 = m.quant_weight_block128(rand(E, H, I) / I ** 0.5)
    sw13, ss13 = m.quant_weight_block128(rand(2 * I, H) / H ** 0.5)
    sw2, ss2 = m.quant_weight_block128(rand(H, I) / I ** 0.5)
    wr, weight = rand(E, H) / H ** 0.5, 1 + 0.1 * rand(H)
    x, res0 = rand(T, H).bfloat16(), rand(T, H).bfloat16()

    def layer(x, res):
        q, s, n = m.rms_norm_quant_fp8(x, weight, residual=res, return_norm=True)
        routed = m.fused_moe(n, w13, w2, n.float() @ wr.t(), 2, True, use_fp8_w8a8=True, w1_scale=s13, w2_scale=s2, block_shape=[128, 128])
        return routed, m.fp8_gated_mlp(q, sw13, ss13, sw2, ss2, x_scale=s, addend=routed)

    res = res0.clone()
    routed, out = layer(x, res)
    h = (x.float() + res0.float()).bfloat16()
    assert torch.equal(res, h)
    hd = h.double()
    y = hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-6) * weight.double()

    def wv(q, s):
        return q.double() * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)

    a, b = (y @ wv(sw13, ss13).t()).chunk(2, 1)
    act = torch.nn.functional.silu(a) * b
    shared = act @ wv(sw2, ss2).t()
    # half a step of e4m3 at most on each of the two quantised operands (the first one's passes through a product and the activation,
    # |act'| < 1.13), and the rounding to bf16
    ya, wa = y.abs() * 2.0 ** -4, wv(sw13, ss13).abs()
    ea, eb = (ya @ wa.t()).chunk(2, 1)
    eh = 1.13 * ea * (b.abs() + eb) + a.abs() * eb
    eh = eh + (act.abs() + eh) * 2.0 ** -4
    allowed = (eh @ wv(sw2, ss2).abs().t()) * 1.01 + (shared.abs() + routed.double().abs()) * 2.0 ** -7 + 1e-3
    assert ((out.double() - routed.double() - shared).abs() <= allowed).all()
    assert float((out.double() - routed.double() - shared).norm() / shared.norm()) < 2.0 ** -4

    xs, rs = x.clone(), res0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(xs, rs)
    torch.cuda.current_stream().wait_stream(side)
    rs.copy_(res0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, again = layer(xs, rs)
    rs.copy_(res0)
    graph.replay()
    assert torch.equal(again, out) and torch.equal(rs, h)


def test_residual_beside_x():
    """x and residual as halves of one buffer's rows, as one tensor, and as rows of one buffer one apart (refused)."""
    both = torch.randn(9, 2 * 384, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").bfloat16()
    w = torch.ones(384, device="cuda")
    x, r = both[:, :384], both[:, 384:]
    want_r = (x.float() + r.float()).bfloat16()
    want = fg().rms_norm_quant_fp8(want_r, w)
    keep = x.clone()
    q, s = fg().rms_norm_quant_fp8(x, w, residual=r)
    assert torch.equal(r, want_r) and torch.equal(x, keep)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
    same = keep.clone()
    fg().rms_norm_quant_fp8(same, w, residual=same)
    assert torch.equal(same, (keep.float() * 2).bfloat16())
    rows = torch.zeros(9, 384, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="shares memory"):
        fg().rms_norm_quant_fp8(rows[:-1], w, residual=rows[1:])


def test_offsets_beyond_32_bits():
    """2.2 G elements: the last rows are what they are in a call of their own."""
    rows, K = 270000, 8192
    x = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    for a in range(0, rows, 30000):
        x[a : a + 30000].normal_()
    w = torch.ones(K, device="cuda")
    tail = x[-300:].clone()
    q, s = fg().rms_norm_quant_fp8(x, w)
    q2, s2 = fg().rms_norm_quant_fp8(tail, w)
    assert torch.equal(q[-300:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-300:], s2)
