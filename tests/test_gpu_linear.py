"""Dense e4m3 products with block scales (fp8_block_linear, fp8_gated_mlp) against their definition in 64 bits.

Tolerances.  The products of e4m3 values are exact in fp32.  A sum of K of them, times two scales per block of 128, has an error of
at most  (128 * 2^-23 + (K/128 + 16) * 2^-24) * sum |terms|:  128 additions inside a block, each off by at most one unit of a 24-bit
significand whether the tensor core rounds or truncates, one fp32 addition per block, and at most 16 for the join of the cluster, the
product of the scales, bias and addend.  The rounding to bf16 adds 2^-8 of the value.
"""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
GROUP = 128


def fg():
    import flaggems_sglang_b200 as m

    return m


def status():
    from flaggems_sglang_b200 import _C

    _C.check_device_status()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(T, K, seed, wide=True):
    x = torch.randn(T, K, generator=gen(seed), device="cuda")
    if wide:  # groups of very different magnitude
        x *= 10.0 ** torch.randint(-3, 3, (T, K // GROUP, 1), generator=gen(seed + 1), device="cuda").expand(-1, -1, GROUP).reshape(T, K)
    return x


def quant(x):
    """Rows -> e4m3 and scales, by the quantiser's rule, in torch."""
    v = x.float().view(x.shape[0], -1, GROUP)
    s = v.abs().amax(-1).clamp_min(1e-10)
    s = s / torch.full_like(s, 448.0)
    return (v / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(x.shape), s


def weight(N, K, seed):
    nb = -(-N // GROUP)
    w = torch.zeros(nb * GROUP, K, device="cuda")
    w[:N] = torch.randn(N, K, generator=gen(seed), device="cuda") / K ** 0.5
    b = w.view(nb, GROUP, K // GROUP, GROUP)
    b *= 10.0 ** torch.randint(-2, 2, (nb, 1, K // GROUP, 1), generator=gen(seed + 1), device="cuda")
    s = b.abs().amax((1, 3)) / 448.0
    return (b / s[:, None, :, None]).clamp(-448, 448).reshape(nb * GROUP, K)[:N].to(torch.float8_e4m3fn).contiguous(), s.contiguous()


def values(q, s):
    return q.double() * s.double().repeat_interleave(GROUP, 1)


def weight_values(q, s):
    return q.double() * s.double().repeat_interleave(GROUP, 0)[: q.shape[0]].repeat_interleave(GROUP, 1)


def sum_error(K):
    return 128 * 2.0 ** -23 + (K / 128 + 16) * 2.0 ** -24


def check(out, xv, wv, more=None):
    """out against xv wv^T + more, all in 64 bits."""
    y, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if more is not None:
        y, size = y + more.double(), size + more.double().abs()
    off = (out.double() - y).abs()
    allowed = y.abs() * 2.0 ** -8 + size * sum_error(xv.shape[1]) * (1 + 2.0 ** -8)
    assert torch.isfinite(out).all()
    assert (off <= allowed).all(), f"off by {float((off - allowed).max())} more than allowed at {(off > allowed).nonzero()[:4].tolist()}"


@pytest.fixture(params=["auto", "cta 1", "cta 3", "cta 8", "pair 1", "pair 2", "pair 3", "pair 4"])
def kernel(request):
    """Every kernel and split, whatever the library would choose for the shape."""
    from flaggems_sglang_b200 import _C

    if request.param != "auto":
        which, split = request.param.split()
        _C.check(_C.lib().fmoe_debug_linear_kernel(int(which == "pair"), int(split)))
    yield request.param
    _C.check(_C.lib().fmoe_debug_linear_kernel(0, 0))


SHAPES = [
    # T, K, N: single token, one block, ragged widths; every token tile; K that does and does not divide among the CTAs of a tile
    (1, 128, 8), (1, 128, 128), (1, 7168, 2048), (2, 256, 136), (3, 384, 1000), (7, 1152, 576), (15, 2048, 4096), (16, 2048, 264),
    (17, 640, 1048), (31, 4096, 120), (48, 2048, 1024), (63, 896, 392), (64, 1408, 512), (65, 1408, 512), (80, 512, 2112),
    (97, 768, 2048), (127, 1024, 640), (128, 1024, 640), (129, 1024, 640), (200, 7168, 576), (255, 384, 1528), (256, 2048, 1024),
    (257, 2048, 1000), (333, 7168, 1584), (511, 1024, 2048), (513, 640, 1160), (1000, 2048, 1544), (2049, 1280, 1152), (4096, 512, 4096),
]


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_linear(T, K, N, kernel):
    xq, xs = quant(rows(T, K, T + K))
    w, ws = weight(N, K, N)
    out = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
    assert out.shape == (T, N) and out.dtype == torch.bfloat16
    check(out, values(xq, xs), weight_values(w, ws))
    for _ in range(3):
        again = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16)), "the result depends on timing"
    status()


@pytest.mark.parametrize("T,K,N", [(1, 256, 64), (70, 1024, 1000), (300, 896, 1544)])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("addend", [False, True])
@pytest.mark.parametrize("x_dtype", ["bf16", "e4m3"])
def test_linear_extras_and_inputs(T, K, N, bias, addend, x_dtype, kernel):
    x = rows(T, K, 5).bfloat16()
    xq, xs = quant(x)
    w, ws = weight(N, K, 6)
    b = None if bias is None else torch.randn(N, generator=gen(7), device="cuda").to(bias)
    a = torch.randn(T, N, generator=gen(8), device="cuda").bfloat16() if addend else None
    more = (0 if b is None else b.double()) + (torch.zeros(T, N, device="cuda").double() if a is None else a.double())
    args = dict(x=x) if x_dtype == "bf16" else dict(x=xq, x_scale=xs)
    keep = None if a is None else a.clone()
    check(fg().fp8_block_linear(w=w, w_scale=ws, bias=b, addend=a, **args), values(xq, xs), weight_values(w, ws), more)
    assert a is None or torch.equal(a, keep)
    status()


def gate_up(xq, xs, w, ws, activation):
    """The first half of the MLP through its own entry point: (q, scale)."""
    from flaggems_sglang_b200 import _C

    T, K = xq.shape
    I = w.shape[0] // 2
    q = torch.empty(T, I, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(T, I // GROUP, dtype=torch.float32, device="cuda")
    _C.check(_C.lib().fmoe_fp8_gate_up(_C.Fp8Args(
        x_dtype=_C.E4M3, activation=_C.ACTIVATIONS[activation], T=T, K=K, I=I, x=xq.data_ptr(), x_scale=xs.data_ptr(), w=w.data_ptr(),
        w_scale=ws.data_ptr(), out=q.data_ptr(), out_scale=s.data_ptr()), _C.stream_ptr()))
    return q, s


MLP_SHAPES = [(1, 128, 128, 8), (1, 7168, 2048, 7168), (4, 2048, 768, 2048), (16, 512, 384, 136), (33, 1152, 256, 1000), (64, 1024, 512, 512),
              (65, 1024, 512, 512), (97, 2048, 768, 2048), (128, 640, 1408, 264), (200, 896, 640, 1160), (555, 1024, 2048, 1024),
              (1030, 2048, 768, 2048)]


@pytest.mark.parametrize("T,K,I,N", MLP_SHAPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_mlp(T, K, I, N, activation, kernel):
    xq, xs = quant(rows(T, K, 11, wide=False))
    w13, s13 = weight(2 * I, K, 12)
    w2, s2 = weight(N, I, 13)
    xv, wv = values(xq, xs), weight_values(w13, s13)
    gate, up = (xv @ wv.t()).chunk(2, dim=1)
    eg, eu = ((xv.abs() @ wv.abs().t()) * sum_error(K)).chunk(2, dim=1)
    h = (torch.nn.functional.silu(gate) if activation == "silu" else torch.nn.functional.gelu(gate)) * up
    # |act(g)| <= |g| and |act'| < 1.13: what the sums' errors do to h, and 2^-20 for exp, erf and division of the activation
    eh = 1.13 * eg * (up.abs() + eu) + gate.abs() * eu + h.abs() * 2.0 ** -20 + (1.13 * gate.abs() * up.abs()) * 2.0 ** -22
    q, s = gate_up(xq, xs, w13, s13, activation)
    # scale: of the group's largest magnitude; value: half a step of e4m3, 2^-4 of it or 2^-10 (subnormal) times the scale
    top, top_e = (z.view(T, I // GROUP, GROUP).abs().amax(-1) for z in (h, eh))
    want = top.clamp_min(1e-10) / 448
    assert ((s.double() - want).abs() <= top_e / 448 + want * 2.0 ** -23).all()
    sv = s.double().repeat_interleave(GROUP, 1)
    off = (q.double() * sv - h).abs()
    assert (off <= (h.abs() + eh) * 2.0 ** -4 + sv * 2.0 ** -10 + eh + h.abs() * 2.0 ** -22 + sv * 448 * 2.0 ** -22).all()
    out = fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs, activation=activation)
    check(out, values(q, s), weight_values(w2, s2))
    add = torch.randn(T, N, generator=gen(14), device="cuda").bfloat16()
    check(fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs, activation=activation, addend=add), values(q, s), weight_values(w2, s2), add)
    status()


def test_gated_mlp_of_bf16_rows_is_that_of_their_quantised_form():
    for T in (1, 50, 140):
        x = rows(T, 1024, 21).bfloat16()
        xq, xs = quant(x)
        w13, s13 = weight(512, 1024, 22)
        w2, s2 = weight(1024, 256, 23)
        a = fg().fp8_gated_mlp(x, w13, s13, w2, s2)
        b = fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs)
        assert torch.equal(a, b)
    status()


def test_quantised_bf16_rows_are_the_quantisers_for_every_significand():
    """Every significand of a value over every one of the group's largest, 24 exponents apart at most, both signs: the quotients lie halfway
    between two e4m3 values as often as bf16 allows.  Read back through a product with the identity."""
    m = (128 + torch.arange(128, device="cuda")).float() / 128
    rows_ = []
    for d in range(0, 24, 1):
        x = (m[None, :] * 2.0 ** -d).repeat(128, 1)  # row: the largest; column: the value
        x = torch.where(torch.arange(128, device="cuda")[None] % 2 == 1, -x, x)
        big = torch.cat([m[:, None] * 2, x[:, 1:]], 1)  # 2 m is larger than all values of the row
        rows_ += [big, torch.cat([m[:, None] * 2, x[:, :1].expand(-1, 127)], 1)]
    x = torch.cat(rows_).bfloat16()
    assert (x.float().abs().amax(1) == x[:, 0].float()).all()
    eye = torch.eye(128, device="cuda").to(torch.float8_e4m3fn)
    one = torch.ones(1, 1, device="cuda")
    xq, xs = quant(x)
    for scale in (1.0, 2.0 ** -20, 2.0 ** 30):
        a = fg().fp8_block_linear((x.float() * scale).bfloat16(), eye, one)
        b = fg().fp8_block_linear(xq, eye, one, x_scale=xs * scale)
        assert torch.equal(a, b)
    status()


def test_rows_do_not_depend_on_their_neighbours(kernel):
    """A row with NaN or infinity in it, or of zeros, leaves the other rows' bits alone; the rows behind the last are not there."""
    T, K, N = 37, 1024, 520
    xq, xs = quant(rows(T, K, 31))
    w, ws = weight(N, K, 32)
    clean = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
    bad, bad_s = xq.clone(), xs.clone()
    bad.view(torch.uint8)[5, 100] = 0x7F  # NaN
    bad_s[9, 3] = float("inf")
    bad.view(torch.uint8)[12] = 0
    got = fg().fp8_block_linear(bad, w, ws, x_scale=bad_s)
    assert torch.isnan(got[5]).all() and not torch.isfinite(got[9]).any() and (got[12] == 0).all()
    keep = [t for t in range(T) if t not in (5, 9, 12)]
    assert torch.equal(got[keep], clean[keep])
    status()


def test_output_rows_behind_the_last_are_left_alone(kernel):
    """Through the C entry point, into a buffer with rows behind the last token's and a neighbour in front."""
    from flaggems_sglang_b200 import _C

    T, K, N = 21, 512, 200
    xq, xs = quant(rows(T, K, 41))
    w, ws = weight(N, K, 42)
    buf = torch.full((T + 20, N), 7.0, dtype=torch.bfloat16, device="cuda")
    _C.check(_C.lib().fmoe_fp8_linear(_C.Fp8Args(x_dtype=_C.E4M3, T=T, K=K, N=N, x=xq.data_ptr(), x_scale=xs.data_ptr(), w=w.data_ptr(),
                                                 w_scale=ws.data_ptr(), out=buf[10:].data_ptr()), _C.stream_ptr()))
    assert (buf[:10] == 7).all() and (buf[10 + T:] == 7).all()
    assert torch.equal(buf[10:10 + T], fg().fp8_block_linear(xq, w, ws, x_scale=xs))
    status()


def test_strided_and_misaligned_inputs():
    T, K, N = 19, 512, 320
    big = rows(T, 2 * K, 51).bfloat16()
    x = big[:, K:]
    w, ws = weight(N, K, 52)
    want = fg().fp8_block_linear(x.contiguous(), w, ws)
    assert torch.equal(fg().fp8_block_linear(x, w, ws), want)
    odd = torch.empty(T * K + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, K)
    odd.copy_(x)
    assert odd.data_ptr() % 16
    assert torch.equal(fg().fp8_block_linear(odd, w, ws), want)
    wo = torch.empty(N * K + 3, dtype=torch.float8_e4m3fn, device="cuda")[3:].view(N, K)
    wo.copy_(w)
    assert torch.equal(fg().fp8_block_linear(x, wo, ws.t().contiguous().t()), want)


def test_empty_batch():
    w, ws = weight(256, 512, 61)
    w2, s2 = weight(512, 128, 62)
    for x in (torch.empty(0, 512, dtype=torch.bfloat16, device="cuda"),):
        assert fg().fp8_block_linear(x, w, ws).shape == (0, 256)
        assert fg().fp8_gated_mlp(x, w, ws, w2, s2).shape == (0, 512)


def test_graphs_and_streams():
    """Captured calls replayed with new inputs, two graphs in turn, and calls on two streams at once give what eager calls give."""
    T, K, I, N = 24, 1024, 512, 1024
    w13, s13 = weight(2 * I, K, 71)
    w2, s2 = weight(N, I, 72)
    inputs = [rows(T, K, 73 + i, wide=False).bfloat16() for i in range(3)]
    want = [fg().fp8_gated_mlp(x, w13, s13, w2, s2) for x in inputs]
    graphs = []
    for _ in range(2):
        x = inputs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fg().fp8_gated_mlp(x, w13, s13, w2, s2)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fg().fp8_gated_mlp(x, w13, s13, w2, s2)
        graphs.append((g, x, y))
    for i in (1, 2, 0):
        for g, x, y in graphs:
            x.copy_(inputs[i])
            g.replay()
        for g, x, y in graphs:
            assert torch.equal(y, want[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(fg().fp8_gated_mlp(inputs[s], w13, s13, w2, s2))
    torch.cuda.synchronize()
    for s in range(2):
        for y in got[s]:
            assert torch.equal(y, want[s])
    status()


def test_refusals():
    w, ws = weight(256, 512, 81)
    x = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    xq, xs = quant(x)
    lin = fg().fp8_block_linear
    for bad in (dict(x=x[None]), dict(x=x.half()), dict(x=x[:, :500]), dict(x=xq), dict(x=xq, x_scale=xs.double()), dict(x=xq, x_scale=xs[:3]),
                dict(x=x, x_scale=xs), dict(w=w.float()), dict(w=w[:, :384]), dict(w=w[:4], w_scale=ws[:1]), dict(w_scale=ws[:1]),
                dict(w_scale=ws.double()), dict(bias=torch.zeros(255, device="cuda")), dict(bias=torch.zeros(256, dtype=torch.int32, device="cuda")),
                dict(addend=torch.zeros(4, 256, device="cuda")), dict(addend=torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            lin(**{**dict(x=x, w=w, w_scale=ws), **bad})
    with pytest.raises(RuntimeError):
        lin(x.cpu(), w, ws)
    w2, s2 = weight(512, 128, 82)
    mlp = fg().fp8_gated_mlp
    for bad in (dict(activation="relu"), dict(w2=w2[:, :64]), dict(w13=w[:200]), dict(w13=w[:128], w13_scale=ws[:1]), dict(w2_scale=s2[:2]),
                dict(w2=w2[:4], w2_scale=s2[:1])):
        with pytest.raises(ValueError):
            mlp(**{**dict(x=x, w13=w, w13_scale=ws, w2=w2, w2_scale=s2), **bad})


def test_short_and_long_way_from_python_give_the_same(monkeypatch):
    """Usual arguments go through the compiled module, others through ctypes: the same kernels, the same bits."""
    from flaggems_sglang_b200 import _C

    assert _C.host(), "the compiled module is not built"
    T, K, I, N = 9, 512, 256, 328
    x = rows(T, K, 91, wide=False).bfloat16()
    xq, xs = quant(x)
    w, ws = weight(N, K, 92)
    w13, s13 = weight(2 * I, K, 93)
    w2, s2 = weight(N, I, 94)
    b, a = torch.randn(N, generator=gen(95), device="cuda"), torch.randn(T, N, generator=gen(96), device="cuda").bfloat16()

    def results():
        out = []
        for extra in (dict(), dict(bias=b), dict(addend=a), dict(bias=b, addend=a)):
            out += [fg().fp8_block_linear(x, w, ws, **extra), fg().fp8_block_linear(xq, w, ws, x_scale=xs, **extra)]
        for extra in (dict(), dict(addend=a), dict(activation="gelu")):
            out += [fg().fp8_gated_mlp(x, w13, s13, w2, s2, **extra), fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs, **extra)]
        for per_token in (False, True):
            for keep in (False, True):
                r = a[:, :K // 2].contiguous().repeat(1, 2)[:, :K].contiguous() if N >= K // 2 else None
                out += [*(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in fg().rms_norm_quant_fp8(
                    x, torch.ones(K, device="cuda"), residual=r, per_token=per_token, return_norm=keep)), r]
        return out

    short = results()
    monkeypatch.setattr(_C, "_host", False)
    monkeypatch.setattr(_C, "host", lambda: False)
    for s, l in zip(short, results()):
        assert s.dtype == l.dtype and s.shape == l.shape and torch.equal(s, l)
    status()


def test_short_way_leaves_odd_arguments_to_the_long_one():
    from flaggems_sglang_b200 import _C

    host = _C.host()
    w, ws = weight(256, 512, 97)
    x = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(512, device="cuda")
    assert host.linear(x, w, ws, None, None, None).shape == (4, 256)
    for bad in ((x.cpu(), w, ws, None, None, None), (x[:, ::2], w, ws, None, None, None), (x, w[:, :256], ws, None, None, None),
                (x, w, ws.double(), None, None, None), (x, w, ws, ws, None, None), (x[:0], w, ws, None, None, None), (3, w, ws, None, None, None),
                (x, w, ws, None, torch.zeros(256, dtype=torch.bfloat16, device="cuda"), None), (x, w, ws, None, None, x), (x, w)):
        assert host.linear(*bad) is None
    assert host.norm(x, one, 1, None, False, False) is None and host.norm(x, one[:256], 1e-6, None, False, False) is None
    assert host.norm(x.half(), one, 1e-6, None, False, False) is None and host.norm(x, one, 1e-6, x.float(), False, False) is None
    assert len(host.norm(x, one, 1e-6, None, False, True)) == 3
    assert host.mlp(x, w, ws, w, ws, None, 0, None) is None and host.mlp(x, w, ws, w, ws, None, "silu", None) is None


@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("T,K,N", [(1, 128, 64), (1, 7168, 264), (7, 1152, 1000), (16, 4096, 136), (17, 2048, 520), (32, 640, 1000),
                                   (33, 1408, 264), (48, 2048, 1024), (64, 896, 120), (65, 512, 264), (97, 2048, 768), (128, 1024, 640),
                                   (129, 640, 392), (300, 1152, 264)])
def test_rows_quantised_in_the_product(T, K, N, split):
    """bf16 rows that the product quantises itself give the bits that they give behind the quantiser's own launch."""
    from flaggems_sglang_b200 import _C

    x = rows(T, K, 31 * T + K).bfloat16()
    x[T // 2, : GROUP // 2] = 0
    x[T // 3, -GROUP:] = 0
    w, ws = weight(N, K, N + 1)
    I = -(-N // GROUP) * GROUP
    w13, ws13 = weight(2 * I, K, N + 2)
    w2, ws2 = weight(N, I, N + 3)
    addend = torch.randn(T, N, generator=gen(5), device="cuda").bfloat16()
    bias = torch.randn(N, generator=gen(6), device="cuda")
    got = {}
    try:
        for which in (0, 2):
            _C.check(_C.lib().fmoe_debug_linear_kernel(which, split))
            got[which] = [fg().fp8_block_linear(x, w, ws, bias=bias, addend=addend), fg().fp8_gated_mlp(x, w13, ws13, w2, ws2, addend=addend)]
            x2 = x.clone()
            x2[0, 0], x2[-1, -1] = float("inf"), float("nan")
            got[which].append(fg().fp8_block_linear(x2, w, ws))
    finally:
        _C.check(_C.lib().fmoe_debug_linear_kernel(0, 0))
    for a, b in zip(got[0], got[2]):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    q, s = quant(x)
    check(got[2][0], values(q, s), weight_values(w, ws), addend.float() + bias)
    status()


@pytest.mark.parametrize("T,K,N", [(262300, 128, 8200), (270000, 8192, 64)])
def test_offsets_beyond_32_bits(T, K, N):
    """More than 2^31 elements of output, or of input; the last rows, and the rows around element 2^31."""
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda")
    for a in range(0, T, 30000):
        x[a : a + 30000].normal_(generator=gen(a))
    xq, xs = fg().per_token_group_quant_fp8(x)
    del x
    w, ws = weight(N, K, 3)
    out = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
    middle = 2 ** 31 // max(K, N)
    for part in (slice(T - 150, T), slice(middle - 70, middle + 70), slice(0, 50)):
        check(out[part], values(xq[part], xs[part]), weight_values(w, ws))
    status()


@pytest.mark.parametrize("which", [0, 1])
def test_offsets_beyond_32_bits_in_the_mlp(which):
    """The last rows' bits are those of a call of their own, by the same kernel."""
    from flaggems_sglang_b200 import _C

    T, K, I, N = 530000, 256, 128, 4096  # 2.2 G elements of output
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda").normal_(generator=gen(1))
    w13, s13 = weight(2 * I, K, 5)
    w2, s2 = weight(N, I, 6)
    try:
        _C.check(_C.lib().fmoe_debug_linear_kernel(which, 1))
        out = fg().fp8_gated_mlp(x, w13, s13, w2, s2)
        part = slice(T - 130, T)
        assert torch.equal(out[part], fg().fp8_gated_mlp(x[part], w13, s13, w2, s2))
    finally:
        _C.check(_C.lib().fmoe_debug_linear_kernel(0, 0))
    status()


def test_rows_of_nan_are_quantised_as_by_the_quantiser():
    """A group of nothing but NaN has the smallest scale, and its values stay NaN; the other groups' products are lost with it, the other
    rows' are not."""
    x = rows(70, 256, 8, wide=False).bfloat16()
    x[3, :GROUP] = float("nan")
    w, ws = weight(264, 256, 9)
    q, s = fg().per_token_group_quant_fp8(x)
    want = fg().fp8_block_linear(q, w, ws, x_scale=s)
    got = fg().fp8_block_linear(x, w, ws)
    assert torch.isnan(got[3]).all()
    keep = [t for t in range(70) if t != 3]
    assert torch.equal(got[keep], want[keep])


def test_many_and_few_tokens_at_once():
    """Captured calls of every kind (rows quantised in the product, shared tiles, pairs with an addend) replayed on three streams at a time."""
    K, I, N = 1024, 512, 2048
    w13, s13 = weight(2 * I, K, 91)
    w2, s2 = weight(N, I, 92)
    w, ws = weight(N, K, 93)
    calls = []
    for i, T in enumerate((3, 100, 2500)):
        x = rows(T, K, 94 + i, wide=False).bfloat16()
        addend = torch.randn(T, N, generator=gen(97 + i), device="cuda").bfloat16()

        def call(x=x, addend=addend):
            return fg().fp8_gated_mlp(x, w13, s13, w2, s2, addend=fg().fp8_block_linear(x, w, ws, addend=addend))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = call().clone()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        calls.append((g, y, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, _, _, s in calls:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, y, want, _ in calls:
        assert torch.equal(y, want)
    status()
