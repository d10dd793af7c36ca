"""The operators around the attention of one step, as timed cases: block tables and slot maps from request lengths, the residual
addition with a root-mean-square norm and an 8-bit output, the gated activation with the same output, and matrix-vector products
with 4-bit weights.

`run` computes them in elementary torch operations (`own` false) or through the public entry points of
`all_quant_b200.uq_cuda` (`own` true); `exact` computes them again from their definitions in 64 bits.  Formats: 8-bit values are
e4m3 with one power-of-two scale (UE8M0 byte s, 2^(s - 127)) per 32 channels; 4-bit weights are e2m1 codes, two to a byte (low
nibble = even channel), with the same kind of scale, in tiles of 128 rows x 128 channels: codes [tiles, K/128, 128, 64], scales
[tiles, K/128, 128, 4] (what `quantize_on_write` writes into a cache of 128-token pages at head_dim 128).
"""
import random

import torch

own = False

EPS = 1e-6
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _plan(name, B, ctx, new, PAGE=64, lens_seed=7):
    """B requests of ctx = (shortest, longest) tokens; new = (fewest, most) of them added by this step, (0, 0): all of them."""
    case = {"op": "plan", "B": B, "lo": ctx[0], "hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "PAGE": PAGE, "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def _norm(name, R, H, dtype="bf16", residual=True):
    case = {"op": "norm", "R": R, "H": H, "dtype": dtype, "residual": residual}
    return {"name": name, **case} if name else case


def _silu(name, R, F, dtype="bf16"):
    case = {"op": "silu", "R": R, "F": F, "dtype": dtype}
    return {"name": name, **case} if name else case


def _linear(name, M, N, K, x="bf16", out="bf16"):
    """M rows of K channels, as bf16 or as 8-bit values with scales (x = "mx8"), times an [N, K] weight in 4 bits."""
    case = {"op": "linear", "M": M, "N": N, "K": K, "x": x, "out": out}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the smallest step: two short chats, four drafts each; a launch is all there is
        _plan("plan_b2_k4", 2, (777, 1000), (4, 4)),
        # a mixed step of a busy server: decodes next to chunks of prompts, an engine's smallest pages
        _plan("plan_mixed_b300_page16", 300, (64, 16384), (1, 512), PAGE=16),
        # whole prompts packed into one step: every page of them comes from the free list
        _plan("plan_prompts_b64", 64, (1024, 8192), (0, 0)),
        # one token of eight sequences, 64 heads of 128
        _norm("norm_r8_h8192", 8, 8192),
        # a prompt's worth of rows, a row count that is no multiple of anything, the first layer's norm (nothing to add yet)
        _norm("norm_r8191_h4096_fp16", 8191, 4096, dtype="fp16", residual=False),
        # the same with the residual, the largest
        _norm("norm_r16384_h8192", 16384, 8192),
        # eight drafts of eight sequences between the two products of a gated block
        _silu("silu_r64_f32768", 64, 32768),
        # a chunk of a prompt, channels that fill no round number of blocks
        _silu("silu_r5001_f11040", 5001, 11040),
        # one token through a small layer's output projection, 8-bit activations
        _linear("linear_m1_4096_mx8", 1, 4096, 4096, x="mx8"),
        # the fused query, key and value projection (64 + 2 x 8 heads of 128) of eight sequences
        _linear("linear_m8_qkv_bf16", 8, 10240, 8192),
        # a down projection with an odd number of rows behind silu_mul
        _linear("linear_m17_down_mx8", 17, 8192, 32768, x="mx8"),
        # gate and up projections of a verify step (eight drafts of eight sequences), the largest weight
        _linear("linear_m64_gate_up_bf16", 64, 65536, 8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["plan", "norm", "silu", "linear", "linear"])
    if op == "plan":
        B = _log_int(rng, 1, 4096)
        hi = max(2, _log_int(rng, 16, 131072) // max(1, B // 32))
        new = rng.choice([(1, 1), (4, 4), (8, 8), (1, 16), (1, 512), (0, 0)])
        if new[1] > hi or (new == (0, 0) and B * hi > 262144):
            new = (1, 1)
        return _plan(None, B, (max(1, new[1], hi // rng.choice([1, 2, 8, 64])), hi), new, PAGE=rng.choice([16, 32, 48, 64, 128]), lens_seed=rng.randrange(1 << 16))
    if op == "norm":
        H = 32 * _log_int(rng, 2, 512)
        return _norm(None, _log_int(rng, 1, min(65536, 16384 * 8192 // H)), H, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]) if H <= 8192 else "bf16", residual=rng.random() < 0.75)
    if op == "silu":
        F = 32 * _log_int(rng, 2, 1024)
        return _silu(None, _log_int(rng, 1, min(32768, 8192 * 8192 // F)), F, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    M = _log_int(rng, 1, 128)
    K = 32 * _log_int(rng, 4, 1024)
    most = 65536 * 8192 * min(64, 64 * 64 // M) // 64
    return _linear(None, M, _log_int(rng, 64, min(65536, most // K)), K, x=rng.choice(["bf16", "mx8"]), out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lens(case):
    """(tokens stored once the step is in, tokens that the step adds) of every request."""
    r = random.Random(case["lens_seed"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    return lens, [n if case["new_hi"] == 0 else min(n, r.randint(case["new_lo"], case["new_hi"])) for n in lens]


def _pages(case):
    P = case["PAGE"]
    lens, new = _lens(case)
    held = [-(-(n - k) // P) for n, k in zip(lens, new)]
    return held, [-(-n // P) - h for n, h in zip(lens, held)]


def _scale_exponent(amax, top_mantissa, top_exponent):
    """The least E with amax <= top * 2^E, top = top_mantissa * 2^top_exponent, 0.5 <= top_mantissa < 1; -127 for a group of zeros."""
    m, e = torch.frexp(amax)
    E = e - top_exponent + (m > top_mantissa).to(e.dtype)
    return torch.where(amax > 0, E, torch.full_like(E, -127)).clamp(-127, 126)


def _pow2(E):
    """2^E as fp32, -126 <= E <= 127."""
    return ((E.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantize_mx8(y):
    """fp32 [..., n] -> e4m3 codes [..., n], scale bytes [..., n / 32]."""
    g = y.unflatten(-1, (-1, 32))
    E = _scale_exponent(g.abs().amax(-1), 0.875, 9)
    return (g * _pow2(-E).unsqueeze(-1)).to(torch.float8_e4m3fn).flatten(-2), (E + 127).to(torch.uint8)


def _quantize_weight(N, K, g):
    """An [N, K] weight of N(0, 1 / K) with a spread per row, in 4 bits, tiled."""
    tiles, ks = -(-N // 128), -(-K // 128)
    codes = torch.zeros(tiles, ks, 128, 64, dtype=torch.uint8, device="cuda")
    scales = torch.full((tiles, ks, 128, 4), 127, dtype=torch.uint8, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    step = max(1, (1 << 24) // (ks * 128 * 128))
    for t in range(0, tiles, step):
        n = min(N - 128 * t, 128 * step)
        rows = 128 * min(step, tiles - t)
        w = torch.zeros(rows, ks * 128, device="cuda")
        w[:n, :K] = torch.randn(n, K, generator=g, device="cuda") * (K ** -0.5 * torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda")))
        w = w.view(rows, ks * 4, 32)
        E = _scale_exponent(w.abs().amax(-1), 0.75, 3)
        q = w * _pow2(-E).unsqueeze(-1)
        c = (torch.bucketize(q.abs(), edges, out_int32=True).to(torch.uint8) | ((q < 0).to(torch.uint8) << 3)).view(-1, 128, ks, 64, 2)
        codes[t:t + step] = (c[..., 0] | (c[..., 1] << 4)).transpose(1, 2)
        scales[t:t + step] = (E + 127).to(torch.uint8).view(-1, 128, ks, 4).transpose(1, 2)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    if case["op"] == "plan":
        lens, new = _lens(case)
        held, need = _pages(case)
        perm = torch.randperm(sum(held) + sum(need), generator=g, device="cuda").to(torch.int32)
        width = max(h + n for h, n in zip(held, need))
        bt = torch.zeros(case["B"], width, dtype=torch.int32, device="cuda")
        mask = torch.arange(width, device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]
        bt[mask] = perm[:sum(held)]
        st["bt"], st["free"], st["T"] = bt, perm[sum(held):].contiguous(), sum(new)
        st["sl"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["qsl"] = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        return st

    def rows(R, H, dtype, size=1.0):   # a few channels carry most of the energy, as the activations of a trained model do
        chan = torch.exp(0.5 * torch.randn(H, generator=g, device="cuda"))
        return (torch.randn(R, H, generator=g, device="cuda").mul_(chan * size)).to(dtype)

    if case["op"] == "norm":
        dt = DTYPES[case["dtype"]]
        st["x"] = rows(case["R"], case["H"], dt)
        st["r"] = rows(case["R"], case["H"], dt, 4.0) if case["residual"] else None
        st["w"] = (1 + 0.1 * torch.randn(case["H"], generator=g, device="cuda")).to(dt)
    elif case["op"] == "silu":
        st["x"] = rows(case["R"], 2 * case["F"], DTYPES[case["dtype"]], 2.0)
    else:
        st["wc"], st["ws"] = _quantize_weight(case["N"], case["K"], g)
        x = rows(case["M"], case["K"], torch.float32)
        st["x"], st["xs"] = _quantize_mx8(x) if case["x"] == "mx8" else (x.bfloat16(), None)
    return st


# ------------------------------------------------------------------------------------------------------------------- run
def _own(st):
    from all_quant_b200 import uq_cuda
    case = st["case"]
    if case["op"] == "plan":
        slots, taken = uq_cuda.plan_step(st["sl"], st["qsl"], st["bt"], case["PAGE"], st["T"], free_pages=st["free"])
        return {"table": st["bt"], "slots": slots, "taken": taken}
    if case["op"] == "norm":
        codes, scales, s = uq_cuda.rms_norm_mx8(st["x"], st["w"], st["r"], eps=EPS)
        return {"codes": codes, "scales": scales.view(torch.float8_e8m0fnu), "sum": s if st["r"] is not None else None}
    if case["op"] == "silu":
        codes, scales = uq_cuda.silu_mul_mx8(st["x"])
        return {"codes": codes, "scales": scales.view(torch.float8_e8m0fnu)}
    return {"y": uq_cuda.fp4_linear(st["x"], st["wc"], st["ws"], case["N"], scales=st["xs"], out_dtype=DTYPES[case["out"]])}


def _weight(codes, scales, N, K, dtype):
    """The [N, K] weight that the codes and scales stand for."""
    one = torch.tensor(FP4 + tuple(-v for v in FP4), dtype=dtype, device="cuda")
    both = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)   # a byte's two values
    tiles, ks = codes.shape[:2]
    w = both[codes.int()].view(tiles, ks, 128, 4, 32)
    w = w * torch.exp2(scales.to(dtype) - 127).unsqueeze(-1)
    return w.permute(0, 2, 1, 3, 4).reshape(tiles * 128, ks * 128)[:N, :K]


def run(st):
    if own:
        return _own(st)
    case = st["case"]
    if case["op"] == "plan":
        P, bt, sl, qsl, free = case["PAGE"], st["bt"], st["sl"].long(), st["qsl"].long(), st["free"]
        n = qsl[1:] - qsl[:-1]
        held = (sl - n + P - 1) // P
        need = (sl + P - 1) // P - held
        upto = need.cumsum(0)
        page = torch.arange(bt.shape[1], device="cuda")[None]
        at = (upto - need - held)[:, None] + page
        mine = (page >= held[:, None]) & (page < (held + need)[:, None])
        bt.copy_(torch.where(mine, free[at.clamp(0, max(0, len(free) - 1))] if len(free) else bt, bt))
        t = torch.arange(st["T"], device="cuda")
        b = torch.searchsorted(qsl[1:].contiguous(), t, right=True)
        pos = (sl - n - qsl[:-1])[b] + t
        return {"table": bt, "slots": bt[b, pos // P].long() * P + pos % P, "taken": upto[-1:].to(torch.int32)}
    if case["op"] == "norm":
        s = st["x"].float() if st["r"] is None else st["x"].float() + st["r"].float()
        codes, scales = _quantize_mx8(s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS) * st["w"].float())
        return {"codes": codes, "scales": scales.view(torch.float8_e8m0fnu), "sum": None if st["r"] is None else s.to(st["x"].dtype)}
    if case["op"] == "silu":
        gate, up = st["x"].float().chunk(2, -1)
        codes, scales = _quantize_mx8(gate / (1 + torch.exp(-gate)) * up)
        return {"codes": codes, "scales": scales.view(torch.float8_e8m0fnu)}
    x = st["x"].float()
    if st["xs"] is not None:
        x = (x.unflatten(-1, (-1, 32)) * torch.exp2(st["xs"].float() - 127).unsqueeze(-1)).flatten(-2)
    return {"y": (x @ _weight(st["wc"], st["ws"], case["N"], case["K"], torch.float32).T).to(DTYPES[case["out"]])}


# ----------------------------------------------------------------------------------------------------------------- exact
def _e4m3(v):
    """Doubles rounded to the nearest e4m3 value, ties to the even one."""
    e = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_mx8(y):
    g = y.reshape(y.shape[0], -1, 32)
    top = g.abs().amax(-1)
    E = torch.ceil(torch.log2(top / 448))
    E = torch.where(torch.ldexp(torch.full_like(E, 448.0), E - 1) >= top, E - 1, torch.where(torch.ldexp(torch.full_like(E, 448.0), E) < top, E + 1, E))
    E = torch.where(top > 0, E, torch.full_like(E, -127.0)).clamp(-127, 126)
    one = torch.ones_like(E)
    return _e4m3(g * torch.ldexp(one, -E).unsqueeze(-1)).reshape(y.shape), torch.ldexp(one, E)


def exact(case, seed):
    if case["op"] == "plan":
        return None   # whole numbers: equal or wrong
    st = prepare(case, seed)
    if case["op"] in ("norm", "silu"):
        parts = {"codes": [], "scales": [], "sum": []}
        for i in range(0, st["x"].shape[0], 2048):
            x = st["x"][i:i + 2048].double()
            if case["op"] == "silu":
                gate, up = x[:, :case["F"]], x[:, case["F"]:]
                y = gate * up / (1 + torch.exp(-gate))
            else:
                x = x if st["r"] is None else x + st["r"][i:i + 2048].double()
                y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * st["w"].double()
                parts["sum"].append(x.float())   # (of two 16-bit values; 32-bit inputs: rounded as their sum is)
            c, s = _exact_mx8(y)
            parts["codes"].append(c.to(torch.float32))   # (e4m3 values and powers of two: exact in 32 bits)
            parts["scales"].append(s.to(torch.float32))
        out = {"codes": torch.cat(parts["codes"]), "scales": torch.cat(parts["scales"])}
        if case["op"] == "norm":
            out["sum"] = None if st["r"] is None else torch.cat(parts["sum"])
        return out
    x, M, N, K = st["x"].double(), case["M"], case["N"], case["K"]
    if st["xs"] is not None:
        x = (x.view(M, -1, 32) * torch.ldexp(torch.ones(M, K // 32, 1, dtype=torch.float64, device="cuda"), st["xs"].double().unsqueeze(-1) - 127)).view(M, K)
    values = torch.tensor(FP4 + tuple(-v for v in FP4), dtype=torch.float64, device="cuda")
    y = torch.empty(M, N, dtype=torch.float64, device="cuda")
    step = 16
    for t in range(0, st["wc"].shape[0], step):
        c = st["wc"][t:t + step].permute(0, 2, 1, 3).reshape(-1, st["wc"].shape[1] * 64).int()   # rows x bytes
        w = torch.empty(c.shape[0], c.shape[1] * 2, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = values[c & 15], values[c >> 4]
        s = st["ws"][t:t + step].permute(0, 2, 1, 3).reshape(c.shape[0], -1).double() - 127
        w = w.view(c.shape[0], -1, 32).mul_(torch.ldexp(torch.ones_like(s), s).unsqueeze(-1)).view(c.shape[0], -1)
        n = min(N - 128 * t, w.shape[0])
        y[:, 128 * t:128 * t + n] = x @ w[:n, :K].T
    return {"y": y}


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "plan":
        taken, tokens, B = sum(_pages(case)[1]), sum(_lens(case)[1]), case["B"]
        return {"bytes": 4 * B + 4 * (B + 1) + 4 * B + 8 * taken + 8 * tokens + 4, "flops": 0}
    if case["op"] == "norm":
        R, H, e = case["R"], case["H"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": R * H * (e * (3 if case["residual"] else 1) + 1) + R * H // 32 + H * e, "flops": 6 * R * H}
    if case["op"] == "silu":
        R, F, e = case["R"], case["F"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": R * F * (2 * e + 1) + R * F // 32, "flops": 6 * R * F}
    M, N, K = case["M"], case["N"], case["K"]
    x = M * K + M * K // 32 if case["x"] == "mx8" else 2 * M * K
    return {"bytes": N * K // 2 + N * K // 32 + x + M * N * (4 if case["out"] == "fp32" else 2), "flops": 2 * M * N * K}
