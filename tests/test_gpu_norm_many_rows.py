"""rms_norm_quant_fp8 where it has many rows: the kernel whose rows arrive in a ring of shared memory (more than 296 bf16 rows of more than
6144 channels with a residual, of more than 7168 without), and the kernels of three CTAs an SM (without a residual, up to 7168 channels, fp32
above 4096).  Against the definition in 64 bits, with the tolerances of test_gpu_norm.py, which hold for any number of rows: a thread adds at
most 16 squares here, too."""
import pytest
import torch

from tests.test_gpu_norm import check, fg, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    from flaggems_sglang_b200 import _C

    yield
    _C.check_device_status()


def both(x, w, residual, per_token, eps=1e-6):
    """The call with and without its norm, each on a residual of its own: (results with norm, residual after)."""
    keep = x.clone()
    r1, r2 = (None if residual is None else residual.clone() for _ in range(2))
    got = fg().rms_norm_quant_fp8(x, w, eps, residual=r1, per_token=per_token, return_norm=True)
    q, s = fg().rms_norm_quant_fp8(x, w, eps, residual=r2, per_token=per_token)
    assert torch.equal(q.view(torch.uint8), got[0].view(torch.uint8)) and torch.equal(s, got[1])
    assert torch.equal(x, keep) and (residual is None or torch.equal(r1, r2))
    return got, r1


# one row more than the line, rounds that end in the middle, CTAs that go round their ring several times; every number of threads' kernel
@pytest.mark.parametrize("rows,K", [(297, 7168), (300, 7296), (2100, 7168), (443, 7680), (1500, 8320), (299, 9216), (1200, 9728), (600, 12288),
                                    (310, 12416), (700, 16384), (8192, 7424)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("per_token", [False, True])
def test_long_bf16_rows(rows, K, residual, per_token):
    x, r, w = make(rows, K, torch.bfloat16, rows + K, residual)
    got, after = both(x, w, r, per_token)
    check(x, w, 1e-6, r, per_token, got, after)


@pytest.mark.parametrize("rows,K", [(900, 6152), (3000, 7176), (445, 8200), (350, 10008), (297, 16376)])
@pytest.mark.parametrize("residual", [False, True])
def test_long_bf16_rows_of_odd_length(rows, K, residual):
    x, r, w = make(rows, K, torch.bfloat16, K, residual)
    got, after = both(x, w.bfloat16(), r, True, 1e-5)
    check(x, w.bfloat16(), 1e-5, r, True, got, after)


@pytest.mark.parametrize("rows,K", [(297, 4224), (700, 5120), (5000, 7168), (444, 2048), (300, 8192)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("per_token", [False, True])
def test_fp32_rows(rows, K, residual, per_token):
    x, r, w = make(rows, K, torch.float32, rows + K, residual)
    got, after = both(x, w, r, per_token)
    check(x, w, 1e-6, r, per_token, got, after)


@pytest.mark.parametrize("K", [7168, 9984, 16384])
def test_strided_rows(K):
    """x and residual as parts of wider rows, as halves of one buffer's rows, and as one tensor."""
    rows = 500
    big, _, w = make(rows, 2 * K + 64, torch.bfloat16, K, False)
    x = big[:, 8 : K + 8]
    w = w[:K]
    store = big[:, K + 16 :].contiguous()
    r = store[:, 8 : K + 8]
    before, outside = r.clone(), store[:, K + 8 :].clone()
    got = fg().rms_norm_quant_fp8(x, w, residual=r, return_norm=True)
    check(x, w, 1e-6, before, False, got, r)
    assert torch.equal(store[:, K + 8 :], outside)
    check(x, w, 1e-6, None, True, fg().rms_norm_quant_fp8(x, w, per_token=True, return_norm=True), None)
    pair = big[:, : 2 * K].contiguous()
    x, r = pair[:, :K], pair[:, K:]
    keep, before = x.clone(), r.clone()
    got = fg().rms_norm_quant_fp8(x, w, residual=r, return_norm=True)
    check(keep, w, 1e-6, before, False, got, r)
    assert torch.equal(x, keep)
    same = keep.clone()
    got = fg().rms_norm_quant_fp8(same, w, residual=same, return_norm=True)
    check(keep, w, 1e-6, keep, False, got, same)


@pytest.mark.parametrize("K", [7296, 9728, 16384])
def test_rows_with_nan_or_infinity_leave_the_others_alone(K):
    rows = 900
    x, r, w = make(rows, K, torch.bfloat16, K, True)
    clean_r = r.clone()
    clean = fg().rms_norm_quant_fp8(x, w, residual=clean_r, return_norm=True)
    bad = x.clone()
    bad[5, 100], bad[500, 3], bad[899, K - 1], bad[296] = float("nan"), float("inf"), float("-inf"), 0
    bad_r = r.clone()
    bad_r[296] = 0
    q, s, n = fg().rms_norm_quant_fp8(bad, w, residual=bad_r, return_norm=True)
    assert torch.isnan(n[5]).all() and torch.isnan(n[500, 3]) and torch.isnan(n[899, K - 1])
    assert (n[296] == 0).all() and (q[296].float() == 0).all()
    keep = [t for t in range(rows) if t not in (5, 296, 500, 899)]
    for a, b in zip((q.view(torch.uint8), s, n, bad_r), (clean[0].view(torch.uint8), clean[1], clean[2], clean_r)):
        assert torch.equal(a[keep], b[keep])


def test_captured_and_on_two_streams():
    rows, K = 700, 7168
    x, r, w = make(rows, K, torch.bfloat16, 5, True)
    after = r.clone()
    want = fg().rms_norm_quant_fp8(x, w, residual=after, return_norm=True)
    calls = []
    for _ in range(2):
        xs, rs = torch.zeros_like(x), torch.zeros_like(r)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fg().rms_norm_quant_fp8(xs, w, residual=rs, return_norm=True)
        calls.append((graph, xs, rs, out, torch.cuda.Stream()))
    for graph, xs, rs, out, stream in calls:
        xs.copy_(x)
    for _ in range(10):
        for graph, xs, rs, out, stream in calls:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                rs.copy_(r)
                graph.replay()
    torch.cuda.synchronize()
    for graph, xs, rs, out, stream in calls:
        assert torch.equal(rs, after)
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("residual", [False, True])
def test_offsets_beyond_32_bits(residual):
    """2.2 G elements: the last rows, those around element 2^31 and the first."""
    rows, K = 264000, 8320
    x = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    for a in range(0, rows, 30000):
        x[a : a + 30000].normal_(generator=torch.Generator(device="cuda").manual_seed(a))
    w = 1 + 0.1 * torch.randn(K, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    middle = 2 ** 31 // K
    parts = [slice(rows - 300, rows), slice(middle - 100, middle + 100), slice(0, 100)]
    r = x.flip(0) if residual else None
    before = [r[p].clone() if residual else None for p in parts]
    q, s, n = fg().rms_norm_quant_fp8(x, w, residual=r, return_norm=True)
    for p, b in zip(parts, before):
        check(x[p], w, 1e-6, b, False, (q[p], s[p], n[p]), r[p] if residual else None)
