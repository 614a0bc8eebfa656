"""Rows of rms_norm_quant_fp8 of either kind of scale are the grouped GEMMs' input as it stands: fmoe_gemm2 of one expert.

Tolerance: products of e4m3 values are exact, each of K additions is off by at most one unit of a 24-bit significand of what has been added up
(2^-23 of the sum of the terms' magnitudes), the scales' two products by 2^-24 each; the rounding to bf16 adds 2^-8 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("per_token", [False, True])
def test_norm_rows_in_the_grouped_gemm(T, per_token):
    import flaggems_sglang_b200 as fg
    from flaggems_sglang_b200 import _C
    from flaggems_sglang_b200.ops.fused_moe import _gemm_args

    K, n = 1024, 512
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    q, s = fg.rms_norm_quant_fp8(x, 1 + 0.1 * torch.randn(K, generator=g, device="cuda"), per_token=per_token)
    w, ws = (fg.quant_weight_per_channel if per_token else fg.quant_weight_block128)(torch.randn(1, n, K, generator=g, device="cuda") / K ** 0.5)
    sorted_ids, expert_ids, num_post = fg.moe_align_block_size(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 128, 1)
    cap = sorted_ids.numel()
    a, a_scale = torch.zeros(cap, K, dtype=torch.uint8, device="cuda"), torch.zeros(cap, *s.shape[1:], device="cuda")
    a[:T], a_scale[:T] = q.view(torch.uint8), s
    out = torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
    _C.check(_C.lib().fmoe_gemm2(_gemm_args(
        variant=_C.VARIANTS["tcgen05"], num_experts=1, top_k=1, block_size=128, numel=T, sorted_cap=cap, max_blocks=cap // 128,
        sorted_token_ids=sorted_ids.data_ptr(), expert_ids=expert_ids.data_ptr(), num_tokens_post_padded=num_post.data_ptr(), dtype=_C.E4M3,
        out_dtype=_C.BF16, n=n, k=K, a_rows=cap, a=a.data_ptr(), w=w.data_ptr(), out=out.data_ptr(), a_scale=a_scale.data_ptr(),
        w_scale=ws.data_ptr(), scale_mode=_C.SCALE_CHANNEL if per_token else _C.SCALE_BLOCK128), _C.stream_ptr()))
    _C.check_device_status()
    if per_token:
        xv, wv = q.double() * s.double()[:, None], w[0].double() * ws[0].double()[:, None]
    else:
        xv = q.double() * s.double().repeat_interleave(128, 1)
        wv = w[0].double() * ws[0].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    y, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    assert ((out.double() - y).abs() <= y.abs() * 2.0 ** -8 + size * (K * 2.0 ** -23 + 2.0 ** -23)).all()
