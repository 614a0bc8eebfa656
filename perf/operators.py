"""What a decoder layer with e4m3 block-scaled weights computes beside its routed experts, as cases that can be timed:

  norm    rms_norm_quant_fp8: the residual's addition, the root-mean-square norm and its e4m3 output with scales (one per
          128 channels, or one per token), with the norm itself where the router reads it
  linear  fp8_block_linear: y = x W^T, W e4m3 with a scale per 128 x 128 block, x e4m3 with a scale per 128 channels (given so,
          or bf16 and quantised in the call), plus a bias or a tensor that joins the sum
  mlp     fp8_gated_mlp: act(x Wg^T) * (x Wu^T) Wd^T, the shared expert (or a dense layer's block), whose output joins the
          routed experts' (`addend`)

`own = False`: each operator in its plain form, elementary torch operations in 32 bits.  `own = True`: the package's operators.
"""
import math

import torch

own = False

GROUP = 128
E4M3_MAX = 448.0
EPS = 1e-6


def _norm(name, T, H, scales="group", x="bf16", residual=True, keep=True):
    return dict(name=name, op="norm", T=T, H=H, scales=scales, x=x, residual=residual, keep=keep)


def _linear(name, T, K, N, x="e4m3", extra="none"):
    return dict(name=name, op="linear", T=T, K=K, N=N, x=x, extra=extra)


def _mlp(name, T, H, I, x="e4m3", addend=True, activation="silu"):
    return dict(name=name, op="mlp", T=T, H=H, I=I, x=x, addend=addend, activation=activation)


def listed():
    return [
        # one decoded token between attention and the experts: a few KB, latency is all there is
        _norm("norm decode 1", 1, 7168),
        # a ragged decode batch of a layer with per-channel weights (one scale per token), rows that no power of two divides
        _norm("norm channel 77", 77, 2880, scales="token", keep=False),
        # a prefill chunk kept in 32 bits, no residual (the first norm of a stack)
        _norm("norm f32 1501", 1501, 4096, x="f32", residual=False, keep=False),
        # prefill: the largest
        _norm("norm prefill 8192", 8192, 7168),
        # one decoded token: the weights are read once, nothing else counts
        _linear("linear decode 1", 1, 7168, 2048),
        # a decode batch that joins the residual, bf16 rows quantised in the call
        _linear("linear decode 48 bf16", 48, 2048, 7168, x="bf16", extra="addend"),
        # a chunk of mixed prefill and decode, an output width that ends inside a weight block, with a bias
        _linear("linear 333 ragged", 333, 7168, 1584, extra="bias"),
        # prefill: the largest
        _linear("linear prefill 8192", 8192, 7168, 4096),
        # the shared expert at one decoded token
        _mlp("mlp decode 1", 1, 7168, 2048),
        # a decode batch of small rows, bf16 in, gelu
        _mlp("mlp decode 97 gelu", 97, 2048, 768, x="bf16", addend=False, activation="gelu"),
        # an odd chunk
        _mlp("mlp 555", 555, 7168, 2048),
        # the shared expert of a prefill chunk
        _mlp("mlp prefill 4096", 4096, 7168, 2048, x="bf16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["norm", "linear", "linear", "mlp"])
    if op == "norm":
        scales = rng.choice(["group", "group", "token"])
        H = 128 * rng.randint(4, 56) if scales == "group" else 8 * rng.randint(64, 896)
        c = _norm("", spread(1, 8192), H, scales, rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.75, rng.random() < 0.5)
        if c["x"] == "f32":
            c["T"] = min(c["T"], 4096)
    elif op == "linear":
        K, N = 128 * rng.randint(4, 56), 16 * rng.randint(8, 448)
        T = min(spread(1, 8192), 8192 * 7168 * 4096 // (K * N))
        c = _linear("", T, K, N, rng.choice(["e4m3", "e4m3", "bf16"]), rng.choice(["none", "none", "bias", "addend"]))
    else:
        H, I = 128 * rng.randint(8, 56), 128 * rng.randint(2, 32)
        T = min(spread(1, 4096), 4096 * 7168 * 2048 // (H * I))
        c = _mlp("", T, H, I, rng.choice(["e4m3", "bf16"]), rng.random() < 0.6, rng.choice(["silu", "silu", "gelu"]))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _weight(gen, N, K):
    """N(0,1)/sqrt(K) in e4m3 with the scale of every 128 x 128 block (the last one of a ragged N holds fewer rows)."""
    nb, kb = -(-N // GROUP), K // GROUP
    w = torch.zeros(nb * GROUP, K, device="cuda")
    w[:N] = torch.randn(N, K, generator=gen, device="cuda") / math.sqrt(K)
    blocks = w.view(nb, GROUP, kb, GROUP)
    scale = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(nb * GROUP, K)[:N]
    return q.to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def _hidden(gen, T, K):
    """Hidden states: N(0,1), and a few channels that are twenty times as large in every token."""
    x = torch.randn(T, K, generator=gen, device="cuda")
    x[:, torch.randint(0, K, (4,), generator=gen, device="cuda")] *= 20.0
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "norm":
        dt = torch.bfloat16 if case["x"] == "bf16" else torch.float32
        s["x"] = _hidden(gen, case["T"], case["H"]).to(dt)
        s["residual"] = (3.0 * _hidden(gen, case["T"], case["H"])).to(dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(case["H"], generator=gen, device="cuda")).to(dt)
        return s
    T = case["T"]
    K, N = (case["K"], case["N"]) if case["op"] == "linear" else (case["H"], case["H"])
    x = _hidden(gen, T, K).bfloat16()
    s["x"], s["x_scale"] = _quant_groups(x.float()) if case["x"] == "e4m3" else (x, None)
    s["bias"] = s["addend"] = None
    if case["op"] == "linear":
        s["w"], s["w_scale"] = _weight(gen, N, K)
        if case["extra"] == "bias":
            s["bias"] = torch.randn(N, generator=gen, device="cuda")
    else:
        s["w13"], s["w13_scale"] = _weight(gen, 2 * case["I"], K)
        s["w2"], s["w2_scale"] = _weight(gen, K, case["I"])
    if case.get("extra") == "addend" or case.get("addend"):
        s["addend"] = torch.randn(T, N, generator=gen, device="cuda").bfloat16()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _to_e4m3(v):
    return v.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _quant_groups(y):
    """fp32 rows -> e4m3 and a scale for each 128 channels: max(amax, 1e-10) / 448."""
    g = y.view(y.shape[0], -1, GROUP)
    amax = g.abs().amax(dim=2).clamp_min(1e-10)
    scale = amax / torch.full_like(amax, E4M3_MAX)
    return _to_e4m3(g / scale[:, :, None]).view(y.shape), scale


def _quant_tokens(y):
    """fp32 rows -> e4m3 and a scale for each row: max(amax / 448, 1 / (448 * 512))."""
    amax = y.abs().amax(dim=1)
    scale = (amax / torch.full_like(amax, E4M3_MAX)).clamp_min(1.0 / (E4M3_MAX * 512.0))
    return _to_e4m3(y / scale[:, None]), scale


def _tokens(s):
    q, scale = (s["x"], s["x_scale"]) if s["x_scale"] is not None else _quant_groups(s["x"].float())
    return _values(q, scale)


def _values(q, scale):
    return (q.float().view(q.shape[0], -1, GROUP) * scale[:, :, None]).view(q.shape)


def _weight_values(w, scale):
    N, K = w.shape
    row = torch.arange(N, device=w.device) // GROUP
    return (w.float().view(N, K // GROUP, GROUP) * scale[row][:, :, None]).view(N, K)


def _act(g, activation):
    if activation == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * 0.70710678118654752))
    return g / (1.0 + torch.exp(-g))


def _finish(y, s):
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["addend"] is not None:
        y = y + s["addend"].float()
    return y.bfloat16()


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        h = s["x"].float()
        out = {}
        if s["residual"] is not None:
            s["residual"].copy_(h + s["residual"].float())
            out["residual"] = s["residual"]
            h = s["residual"].float()
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS) * s["weight"].float()
        out["q"], out["scale"] = _quant_groups(y) if case["scales"] == "group" else _quant_tokens(y)
        if case["keep"]:
            out["norm"] = y.to(s["x"].dtype)
        return out
    if case["op"] == "linear":
        return _finish(_tokens(s) @ _weight_values(s["w"], s["w_scale"]).t(), s)
    gu = _tokens(s) @ _weight_values(s["w13"], s["w13_scale"]).t()
    I = case["I"]
    h = _values(*_quant_groups(_act(gu[:, :I], case["activation"]) * gu[:, I:]))
    return _finish(h @ _weight_values(s["w2"], s["w2_scale"]).t(), s)


def run(s):
    if not own:
        return _plain(s)
    import flaggems_sglang_b200 as fg

    case = s["case"]
    if case["op"] == "norm":
        got = fg.rms_norm_quant_fp8(s["x"], s["weight"], EPS, residual=s["residual"], per_token=case["scales"] == "token",
                                    return_norm=case["keep"])
        out = {"q": got[0], "scale": got[1]}
        if s["residual"] is not None:
            out["residual"] = s["residual"]
        if case["keep"]:
            out["norm"] = got[2]
        return out
    if case["op"] == "linear":
        return fg.fp8_block_linear(s["x"], s["w"], s["w_scale"], x_scale=s["x_scale"], bias=s["bias"], addend=s["addend"])
    return fg.fp8_gated_mlp(s["x"], s["w13"], s["w13_scale"], s["w2"], s["w2_scale"], x_scale=s["x_scale"],
                            activation=case["activation"], addend=s["addend"])


def work(case):
    """Inputs once and outputs once; the products of the matrices."""
    T = case["T"]
    if case["op"] == "norm":
        H, eb = case["H"], 2 if case["x"] == "bf16" else 4
        scales = 4 * (H // GROUP if case["scales"] == "group" else 1)
        rows = eb * H * (1 + 2 * case["residual"] + case["keep"]) + H + scales
        return {"bytes": T * rows + eb * H, "flops": 6 * T * H}
    K, N = (case["K"], case["N"]) if case["op"] == "linear" else (case["H"], case["H"])
    x = T * (2 * K if case["x"] == "bf16" else K + K // GROUP * 4)

    def weight(n, k):
        return n * k + -(-n // GROUP) * (k // GROUP) * 4

    if case["op"] == "linear":
        extra = {"none": 0, "bias": 4 * N, "addend": 2 * T * N}[case["extra"]]
        return {"bytes": x + weight(N, K) + extra + 2 * T * N, "flops": 2 * T * N * K}
    I = case["I"]
    return {"bytes": x + weight(2 * I, K) + weight(K, I) + 2 * T * K * (1 + case["addend"]), "flops": 6 * T * K * I}


# ---- the same from the definitions in 64 bits --------------------------------------------------------------------------

def _round_e4m3_64(v):
    """Nearest e4m3 value (ties to even): steps of 2^(e-3) between 2^e and 2^(e+1), of 2^-9 below 2^-6, at most 448."""
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _expand(scale, rows, cols):
    """Scales of blocks (of `rows` x 128 each) -> one per value."""
    return scale.double().repeat_interleave(rows, dim=0).repeat_interleave(GROUP, dim=1)[:, :cols]


def _rows_64(y):
    """What rows quantised by groups stand for.  The scale and the quotient are 32-bit numbers by the quantiser's definition:
    quotients of two bf16 values often lie halfway between two e4m3 values, and that rounding makes them a tie."""
    amax = torch.clamp(y.reshape(-1, GROUP).abs().max(dim=1).values, min=1e-10)
    scale = (amax / E4M3_MAX).float().double()
    quotient = (y.reshape(-1, GROUP) / scale[:, None]).float().double()
    return (_round_e4m3_64(quotient) * scale[:, None]).reshape(y.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    T = case["T"]
    if case["op"] == "norm":
        h, out = x, {}
        if case["residual"]:
            h = (x + s["residual"].double()).to(s["x"].dtype).double()  # the norm is of what the residual holds from here on
            out["residual"] = h
        y = h * s["weight"].double()[None, :] * torch.rsqrt(h.pow(2).mean(dim=1) + EPS)[:, None]
        if case["scales"] == "group":
            out["scale"] = torch.clamp(y.reshape(T, -1, GROUP).abs().max(dim=2).values, min=1e-10) / E4M3_MAX
            out["q"] = (y.reshape(T, -1, GROUP) / out["scale"].unsqueeze(2)).reshape(T, -1)  # before its rounding to e4m3
        else:
            out["scale"] = torch.clamp(y.abs().max(dim=1).values / E4M3_MAX, min=1.0 / (E4M3_MAX * 512.0))
            out["q"] = y / out["scale"].unsqueeze(1)
        if case["keep"]:
            out["norm"] = y
        return out
    K = x.shape[1]
    xv = x * _expand(s["x_scale"], 1, K) if case["x"] == "e4m3" else _rows_64(x)

    def product(a, w, scale):
        return torch.einsum("tk,nk->tn", a, w.double() * _expand(scale, GROUP, w.shape[1])[: w.shape[0]])

    if case["op"] == "linear":
        y = product(xv, s["w"], s["w_scale"])
    else:
        gate, up = product(xv, s["w13"], s["w13_scale"]).chunk(2, dim=1)
        phi = torch.special.ndtr(gate) if case["activation"] == "gelu" else torch.sigmoid(gate)
        y = product(_rows_64(gate * phi * up), s["w2"], s["w2_scale"])
    for more in ("bias", "addend"):
        if s[more] is not None:
            y = y + s[more].double()
    return y
