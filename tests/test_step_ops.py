"""The operators around a layer's attention - plan_step, rms_norm_mx8, silu_mul_mx8, fp4_linear - against plain implementations in
64 bits (numpy), their refusals, and a layer's step made of them.

Tolerances.  A rounding to e4m3 is off by at most half a step: 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it.  The
value that is rounded carries an fp32 error: sums of at most 32768 squares as a tree of 8 + log2 stages, a reciprocal root (2 ulp),
three products, an exponential (2 ulp) - under 32 roundings of 2^-24, taken as YERR = 2^-19 of the value.  So a code has to be
one that some y within (1 +- YERR) of the 64-bit value rounds to, and a scale one that some such maximum asks for."""
import ctypes

import numpy as np
import pytest
import torch

from all_quant_b200 import uq_cuda, vllm_adapter

YERR = 2.0 ** -19
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
FP4 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


# ---------------------------------------------------------------------------------------------------- plain forms, 64 bits
def e4m3(v):
    """Nearest e4m3 value, ties to even."""
    v = np.asarray(v, np.float64)
    e = np.maximum(np.frexp(v)[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.clip(np.rint(v / step) * step, -448, 448)


def exponent(amax):
    """The least E with amax <= 448 * 2^E, -127 for zero."""
    m, e = np.frexp(np.asarray(amax, np.float64))
    return np.where(amax > 0, np.maximum(e - 9 + (m > 0.875), -127), -127)


def check_mx8(codes, scales, y):
    """codes e4m3 tensor [..., n], scales uint8 [..., n/32] against the 64-bit rows y."""
    y = np.asarray(y, np.float64)
    got = codes.float().cpu().numpy().astype(np.float64).reshape(-1, 32)
    E = scales.cpu().numpy().astype(np.int64).reshape(-1) - 127
    g = y.reshape(-1, 32)
    amax = np.abs(g).max(1)
    assert (E >= exponent(amax * (1 - YERR))).all() and (E <= exponent(amax * (1 + YERR))).all()
    scaled = np.ldexp(g, -E[:, None])
    a, b = e4m3(scaled * (1 - YERR)), e4m3(scaled * (1 + YERR))
    assert ((got >= np.minimum(a, b)) & (got <= np.maximum(a, b))).all()
    assert (np.abs(np.ldexp(got, E[:, None]) - g) <= (2.0 ** -4 + YERR) * np.abs(g) + np.ldexp(2.0 ** -10, E)[:, None]).all()


def weight64(wc, ws, n, K):
    c, s = wc.cpu().numpy(), ws.cpu().numpy().astype(np.int64)
    tiles, ks = c.shape[:2]
    w = np.stack([FP4[c & 15], FP4[c >> 4]], -1).reshape(tiles, ks, 128, 4, 32)
    w = np.ldexp(w, (s - 127)[..., None])
    return w.transpose(0, 2, 1, 3, 4).reshape(tiles * 128, ks * 128)[:n, :K]


def mx8_values(codes, scales):
    c = codes.float().cpu().numpy().astype(np.float64)
    s = scales.cpu().numpy().astype(np.int64) - 127
    return np.ldexp(c.reshape(s.shape + (32,)), s[..., None]).reshape(c.shape)


def check_linear(got, x64, w64, dtype, split=False):
    """fp32 sums of exact products, in any order of blocks of 32: every partial sum is at most A = sum |x w|, every one of the
    K / 32 + 32 additions on the way to an output off by at most 2^-22 of that; then one rounding to the output's type.  Rows
    split from bf16: what lies under 2^-21 of a group's largest value is lost."""
    y, A = x64 @ w64.T, np.abs(x64) @ np.abs(w64).T
    K = x64.shape[1]
    tol = (K / 32 + 32) * 2.0 ** -22 * A + torch.finfo(dtype).eps / 2 * np.abs(y) + torch.finfo(dtype).tiny
    if split:
        top = np.abs(x64).reshape(-1, K // 32, 32).max(2).repeat(32, 1)
        tol = tol + 2.0 ** -21 * top @ np.abs(w64).T
    assert (np.abs(got.double().cpu().numpy() - y) <= tol).all()


def plan64(lens, new, table, page, T, free=None, starts=None):
    """One request and one token at a time."""
    table, slots, taken = table.copy(), np.full(T, -1, np.int64), 0
    first = 0
    for b, (n, k) in enumerate(zip(lens, new)):
        n = max(n, 0)
        k = max(k, 0)
        mp = table.shape[1]
        held = min(-(-max(n - k, 0) // page), mp)
        if free is not None:
            for j in range(held, min(-(-n // page), mp)):
                table[b, j] = free[taken] if taken < len(free) else -1
                taken += 1
        at = first if starts is None else starts[b]
        for i in range(k):
            p = n - k + i
            if 0 <= p and at + i < T and p // page < mp and table[b, p // page] >= 0:
                slots[at + i] = int(table[b, p // page]) * page + p % page
        first += k
    return table, slots, taken


# ------------------------------------------------------------------------------------------------------- refusals (CPU)
FAKE = 0x7F0000000000


def _p(i, delta=0):
    return ctypes.c_void_p(FAKE + i * 0x1000000 + delta)


@pytest.mark.parametrize("over", [dict(B=-1), dict(B=16385), dict(K=-1), dict(T=-1), dict(T=1 << 31), dict(PAGE=0), dict(max_pages=-1), dict(stride=7),
                                  dict(n_free=-1), dict(lens=None), dict(table=None), dict(slots=None), dict(n_free=4, taken=None), dict(n_free=4, free=None),
                                  dict(B=16384, max_pages=1 << 18, stride=1 << 18), dict(K=2, starts=_p(1))])
def test_plan_refuses(over):
    a = dict(lens=_p(0), starts=None, K=1, table=_p(2), stride=8, free=_p(3), n_free=0, slots=_p(4), taken=_p(5), B=4, T=4, PAGE=16, max_pages=8)
    a.update(over)
    L = uq_cuda.lib()
    n0 = L.uqb_launch_count()
    assert L.uqb_plan_step_launch(*[a[k] for k in ("lens", "starts", "K", "table", "stride", "free", "n_free", "slots", "taken", "B", "T", "PAGE", "max_pages")], None) == 1
    assert L.uqb_launch_count() == n0


@pytest.mark.parametrize("over", [dict(H=0), dict(H=48), dict(H=32800), dict(rows=-1), dict(dtype=3), dict(eps=0.0), dict(eps=float("nan")), dict(sum=None), dict(r=None),
                                  dict(x=None), dict(x=_p(0, 8)), dict(w=_p(2, 2)), dict(codes=_p(4, 4)), dict(scales=None), dict(sum=_p(3, 8))])
def test_norm_refuses(over):
    a = dict(x=_p(0), r=_p(1), w=_p(2), sum=_p(3), codes=_p(4), scales=_p(5), rows=4, H=64, dtype=1, eps=1e-6)
    a.update(over)
    L = uq_cuda.lib()
    n0 = L.uqb_launch_count()
    assert L.uqb_rms_norm_mx8_launch(*[a[k] for k in ("x", "r", "w", "sum", "codes", "scales", "rows", "H", "dtype", "eps")], None) == 1
    assert L.uqb_launch_count() == n0


@pytest.mark.parametrize("over", [dict(F=0), dict(F=40), dict(F=(1 << 20) + 32), dict(rows=-1), dict(dtype=-1), dict(x=None), dict(x=_p(0, 2)), dict(codes=_p(1, 4)), dict(scales=None)])
def test_silu_refuses(over):
    a = dict(x=_p(0), codes=_p(1), scales=_p(2), rows=4, F=64, dtype=1)
    a.update(over)
    L = uq_cuda.lib()
    n0 = L.uqb_launch_count()
    assert L.uqb_silu_mul_mx8_launch(*[a[k] for k in ("x", "codes", "scales", "rows", "F", "dtype")], None) == 1
    assert L.uqb_launch_count() == n0


@pytest.mark.parametrize("over", [dict(M=-1), dict(M=(1 << 24) + 1), dict(N=0), dict(K=0), dict(K=48), dict(dtype=3), dict(x=None), dict(wc=None), dict(ws=None), dict(out=None),
                                  dict(x=_p(0, 8)), dict(wc=_p(2, 16)), dict(ws=_p(3, 8)), dict(out=_p(4, 4)), dict(xs=_p(1, 2)), dict(xs=None, scratch=None),
                                  dict(xs=None, scratch=_p(5, 8))])
def test_linear_refuses(over):
    a = dict(x=_p(0), xs=_p(1), wc=_p(2), ws=_p(3), out=_p(4), scratch=_p(5), M=9, N=128, K=64, dtype=1)
    a.update(over)
    L = uq_cuda.lib()
    n0 = L.uqb_launch_count()
    assert L.uqb_fp4_linear_launch(*[a[k] for k in ("x", "xs", "wc", "ws", "out", "scratch", "M", "N", "K", "dtype")], None) == 1
    assert L.uqb_launch_count() == n0


def test_scratch_sizes():
    """Both planes of codes and scales: 16, 32, 64 or 128 rows, or tiles of 128; none up to 4 rows."""
    for M, rows in ((1, 0), (4, 0), (5, 16), (8, 16), (9, 32), (16, 32), (17, 64), (33, 128), (64, 128), (65, 256), (1000, 2048)):
        for K in (32, 96, 8192):
            assert uq_cuda.fp4_linear_scratch_bytes(M, K) == rows * (K + K // 32)
    assert uq_cuda.fp4_linear_scratch_bytes(0, 64) == 0 and uq_cuda.fp4_linear_scratch_bytes(4, 40) == 0


def test_cpu_tensors_are_refused():
    z = torch.zeros
    for call in (lambda: uq_cuda.plan_step(z(2, dtype=torch.int32), 1, z(2, 4, dtype=torch.int32), 16, 2), lambda: uq_cuda.rms_norm_mx8(z(2, 64)),
                 lambda: uq_cuda.silu_mul_mx8(z(2, 64)), lambda: uq_cuda.pack_fp4_weight(z(2, 64)),
                 lambda: uq_cuda.fp4_linear(z(1, 128, dtype=torch.bfloat16), z(1, 1, 128, 64, dtype=torch.uint8), z(1, 1, 128, 4, dtype=torch.uint8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_kernels_keep_the_order_of_dependents():
    """What every kernel launched as a programmatic dependent keeps to (see test_kernel_order.py): it waits before it reads or writes
    global memory, lets its successor in only behind its own wait (but for one), takes tensor memory only there, and asks for the SM count."""
    from tests.test_kernel_order import CSRC, kernels
    import os
    import re
    seen = 0
    for name in ("uq_plan.cu", "uq_rows.cu", "uq_linear.cu"):
        for kernel, body in kernels(name).items():
            seen += 1
            waits = [m.start() for m in re.finditer(r"uq_pdl_wait\(\)", body)]
            assert waits and body.count("uq_pdl_release()") == 1 and "__ldg" not in body, kernel
            # (the first of two waits is that of the early exit on a misplaced buffer)
            assert len(waits) == (2 if "linear" in kernel else 1), kernel
            # (the split of rows, which only the products' kernel of the same call follows, lets that set itself up early)
            assert (body.index("uq_pdl_release()") > waits[-1]) == ("split" not in kernel), kernel
            assert not any(what in body[:waits[-1]] for what in ("tcgen05.alloc", "tma_load", "bulk_load", ".load(", "seq_lens")), kernel
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        assert "__restrict__" not in text and not re.search(r"\b148\b", text), name
    assert seen == 6


# ---------------------------------------------------------------------------------------------------------------- plan
gpu = pytest.mark.gpu


def _plan_case(rng, B, page, lo, hi, new_lo, new_hi, spare=0, extra_cols=0):
    lens = rng.integers(lo, hi + 1, B)
    new = lens.copy() if new_hi < 0 else np.minimum(rng.integers(new_lo, new_hi + 1, B), lens)
    held, total = -(-(lens - new) // page), -(-lens // page)
    perm = rng.permutation(int(total.sum()) + spare).astype(np.int32)
    table = np.full((B, max(int(total.max(initial=0)), 1) + extra_cols), -7, np.int32)
    at = 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    return lens, new, table, perm[at:]


def _run_plan(lens, new, table, page, T, free, mode):
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    bt = dev(table)
    arg = {"starts": dev(starts), "uniform": int(new[0]) if len(new) else 1, "whole": None}[mode]
    slots, taken = uq_cuda.plan_step(dev(lens.astype(np.int32)), arg, bt, page, T, free_pages=None if free is None else dev(free))
    return bt.cpu().numpy(), slots.cpu().numpy(), None if taken is None else int(taken)


@gpu
@pytest.mark.parametrize("B,page,lo,hi,new_lo,new_hi,mode", [
    (1, 64, 1, 1, 1, 1, "uniform"), (2, 64, 777, 1000, 4, 4, "uniform"), (5, 16, 1, 40, 0, 9, "starts"), (300, 16, 64, 1500, 1, 128, "starts"),
    (513, 48, 1, 700, 0, 3, "starts"), (64, 64, 0, 900, 0, -1, "whole"), (3, 1, 0, 50, 0, -1, "whole"), (4096, 128, 1, 300, 1, 1, "uniform"), (16384, 16, 1, 20, 0, 2, "starts")])
def test_plan_matches_the_plain_form(B, page, lo, hi, new_lo, new_hi, mode):
    lens, new, table, free = _plan_case(np.random.default_rng(B), B, page, lo, hi, new_lo, new_hi, spare=3, extra_cols=2)
    if mode == "uniform":
        new[:] = new[0]
        lens = np.maximum(lens, new)
        held = -(-(lens - new) // page)
        total = int((-(-lens // page) - held).sum())
        table = np.full_like(table, -7)
        for b in range(B):
            table[b, :held[b]] = np.arange(held[b]) + 1000 * b
        free = np.random.default_rng(7).permutation(total + 3).astype(np.int32)
    T = int(new.sum()) + 5   # rows behind the last token
    want = plan64(lens, new, table, page, T, free)
    got = _run_plan(lens, new, table, page, T, free, mode)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all() and got[2] == want[2]
    # a complete table: the same slots, nothing written
    again = _run_plan(lens, new, want[0], page, T, None, mode)
    assert (again[0] == want[0]).all() and (again[1] == want[1]).all() and again[2] is None


@gpu
def test_plan_when_pages_run_out_or_the_table_is_too_narrow():
    lens, new, table, free = _plan_case(np.random.default_rng(3), 9, 16, 20, 90, 5, 60)
    for n_free in (0, 1, len(free) // 2):
        want = plan64(lens, new, table, 16, int(new.sum()), free[:n_free])
        got = _run_plan(lens, new, table, 16, int(new.sum()), free[:n_free], "starts")
        assert (got[0] == want[0]).all() and (got[1] == want[1]).all() and got[2] == want[2] > n_free
    narrow = np.ascontiguousarray(table[:, :3])
    want = plan64(lens, new, narrow, 16, int(new.sum()), free)
    got = _run_plan(lens, new, narrow, 16, int(new.sum()), free, "starts")
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all() and got[2] == want[2] and (want[1] == -1).any()


@gpu
def test_plan_odd_inputs():
    # more new tokens than stored ones, a request of length zero, one below zero, starts behind the token axis
    lens, new = np.array([3, 0, -4, 33]), np.array([5, 0, 0, 2])
    table, free = np.full((4, 4), -7, np.int32), np.arange(50, 60, dtype=np.int32)
    table[3, :2] = (8, 9)
    for T in (0, 4, 7, 9):
        want = plan64(lens, new, table, 16, T, free)
        got = _run_plan(lens, new, table, 16, T, free, "starts")
        assert (got[0] == want[0]).all() and (got[1] == want[1]).all() and got[2] == want[2], T
    # no request at all
    got = _run_plan(lens[:0], new[:0], table[:0], 16, 3, free, "starts")
    assert (got[1] == -1).all() and got[2] == 0
    # starts that do not begin at zero, and a strided table inside a wider one whose other rows and columns stay
    big = torch.full((6, 10), -7, dtype=torch.int32, device="cuda")
    bt = big[1:, 2:6]
    bt[0, 0] = 4
    starts = torch.tensor([2, 3, 5], dtype=torch.int32, device="cuda")
    slots, taken = uq_cuda.plan_step(torch.tensor([17, 2], device="cuda"), starts, bt, 16, 6, free_pages=torch.tensor([11, 12], dtype=torch.int32, device="cuda"))
    assert slots.tolist() == [-1, -1, 11 * 16, 12 * 16, 12 * 16 + 1, -1] and int(taken) == 2
    want = torch.full((6, 10), -7, dtype=torch.int32)
    want[1, 2], want[1, 3], want[2, 2] = 4, 11, 12
    assert torch.equal(big.cpu(), want)


@gpu
def test_plan_refuses_in_python():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for kw in (dict(new=0), dict(new=i(5)), dict(bt=i(3, 2).long()), dict(bt=i(1, 2)), dict(page=0), dict(T=-1), dict(free=i(4).long()), dict(free=i(8)[::2]), dict(bt=i(2, 3).t()),
               dict(slots=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        a = dict(new=1, bt=i(2, 2), page=16, T=2, free=None, slots=None, **{}) | kw
        with pytest.raises(RuntimeError):
            uq_cuda.plan_step(i(2), a["new"], a["bt"], a["page"], a["T"], free_pages=a["free"], slots=a["slots"])


# ------------------------------------------------------------------------------------------------------- norm and gate
def _rand(shape, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    return (torch.randn(*shape, generator=g, device="cuda") * chan * size).to(dtype)


def _f64(t):
    return t.double().cpu().numpy()


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,H,residual,weight", [(1, 32, True, True), (3, 64, False, True), (7, 256, True, False), (5, 288, True, True), (130, 512, True, True), (2, 1024, False, False),
                                                 (9, 1056, True, True), (8, 8192, True, True), (3, 11040, True, True), (2, 16384, False, True), (2, 32768, True, True), (700, 4096, True, True)])
def test_norm_matches_the_plain_form(dtype, R, H, residual, weight):
    dt = DT[dtype]
    x, r = _rand((R, H), dt, 1), _rand((R, H), dt, 2, 4.0) if residual else None
    w = (1 + 0.1 * _rand((H,), torch.float32, 3)).to(dt) if weight else None
    codes, scales, s = uq_cuda.rms_norm_mx8(x, w, r, eps=1e-5)
    s64 = _f64(x) + (_f64(r) if residual else 0)
    y = s64 / np.sqrt((s64 ** 2).mean(-1, keepdims=True) + 1e-5) * (_f64(w) if weight else 1)
    check_mx8(codes, scales, y)
    if residual:
        assert (np.abs(_f64(s) - s64) <= (torch.finfo(dt).eps / 2 + 2.0 ** -24) * np.abs(s64) + torch.finfo(dt).tiny).all()
    else:
        assert s is None


@gpu
def test_norm_in_place_strided_and_batched():
    x, r, w = _rand((6, 5, 96), torch.bfloat16, 1), _rand((6, 5, 96), torch.bfloat16, 2), _rand((96,), torch.bfloat16, 3)
    want = uq_cuda.rms_norm_mx8(x, w, r)
    assert want[0].shape == (6, 5, 96) and want[1].shape == (6, 5, 3) and want[2].shape == (6, 5, 96)
    # rows of a wider tensor, a weight off its 16-byte boundary
    wide = torch.zeros(6, 5, 200, dtype=torch.bfloat16, device="cuda")
    wide[..., 3:99] = x
    off = torch.cat([w[:1], w])[1:]
    got = uq_cuda.rms_norm_mx8(wide[..., 3:99], off, r)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    for target in (r, x):   # the sum into the residual's or the input's own memory
        mine = target.clone()
        args = (mine, w, r) if target is x else (x, w, mine)
        got = uq_cuda.rms_norm_mx8(*args, sum_out=mine)
        assert got[2] is mine and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # outputs given: rows behind them stay as they were
    c, s = torch.full((8, 5, 96), 1.0, device="cuda").to(torch.float8_e4m3fn), torch.full((8, 5, 3), 9, dtype=torch.uint8, device="cuda")
    uq_cuda.rms_norm_mx8(x, w, r, codes=c[:6], scales=s[:6])
    assert torch.equal(c[:6].view(torch.uint8), want[0].view(torch.uint8)) and (c[6:].float() == 1).all() and (s[6:] == 9).all() and torch.equal(s[:6], want[1])
    # no rows
    got = uq_cuda.rms_norm_mx8(x[:0], w, r[:0])
    assert got[0].shape == (0, 5, 96)


@gpu
@pytest.mark.parametrize("H", [64, 2048])
def test_norm_extremes(H):
    """Zeros, one large value, groups at and around a scale's border, values whose squares leave fp32, NaN and infinity."""
    x = _rand((9, H), torch.float32, 5)
    x[0] = 0
    x[1] = 0
    x[1, 33] = 1e-3
    x[2] *= 1e25
    x[3] *= 1e-30
    x[4, :32] = 0
    x[5] = 1.0
    x[6] = torch.where(torch.arange(H, device="cuda") % 2 == 0, 3.0e38, -1.0e30)
    x[7, 5] = float("nan")
    x[8, 5] = float("inf")
    w = torch.ones(H, device="cuda")
    w[:32] = 448.0   # x[5]: y = 448 / sqrt(1 + eps), under the border by eps / 2 ~ 2^-11
    codes, scales, _ = uq_cuda.rms_norm_mx8(x, w, eps=1e-3)
    x64 = _f64(x)[:7]
    check_mx8(codes[:7], scales[:7], x64 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + 1e-3) * _f64(w))
    assert (codes[0].float() == 0).all() and (scales[0] == 0).all() and codes[7].float().isnan().all()
    assert codes[8, 5].float().isnan() and (codes[8].float().nan_to_num(0) == 0).all()   # s * (1 / inf)


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,F", [(1, 32), (3, 96), (64, 2048), (5, 2080), (33, 11040), (2, 32768)])
def test_silu_matches_the_plain_form(dtype, R, F):
    x = _rand((R, 2 * F), DT[dtype], R, 3.0)
    codes, scales = uq_cuda.silu_mul_mx8(x)
    g, u = _f64(x)[:, :F], _f64(x)[:, F:]
    check_mx8(codes, scales, g / (1 + np.exp(-g)) * u)


@gpu
def test_silu_extremes():
    g = torch.tensor([0.0, -0.0, 1e-30, -80.0, -87.0, 80.0, 1e20, -60.0], device="cuda").repeat(8).view(1, 64)
    u = torch.tensor([1.0, -1.0, 3.0, 2.0, 5.0, -7.0, 1e5, 1e10], device="cuda").repeat_interleave(8).view(1, 64)
    codes, scales = uq_cuda.silu_mul_mx8(torch.cat([g, u], 1))
    g64, u64 = _f64(g), _f64(u)
    check_mx8(codes, scales, g64 / (1 + np.exp(-g64)) * u64)
    x = torch.ones(2, 128, device="cuda")
    x[0, 3], x[1, 40], x[0, 64 + 50] = float("nan"), float("inf"), float("-inf")
    codes, scales = uq_cuda.silu_mul_mx8(x)
    bad = codes.float().isnan()
    assert bad.sum() == 3 and bad[0, 3] and bad[1, 40] and bad[0, 50]
    assert (codes[0, :32].float()[torch.arange(32) != 3] > 0).all()   # the NaN's neighbours keep their values


@gpu
def test_row_operators_refuse_in_python():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: uq_cuda.rms_norm_mx8(x[:, :48]), lambda: uq_cuda.rms_norm_mx8(x.double()), lambda: uq_cuda.rms_norm_mx8(x, x[0].float()), lambda: uq_cuda.rms_norm_mx8(x, x[0], x[:2]),
                 lambda: uq_cuda.rms_norm_mx8(x, x[0], eps=0), lambda: uq_cuda.rms_norm_mx8(x, x[0], sum_out=x), lambda: uq_cuda.rms_norm_mx8(x, codes=x), lambda: uq_cuda.silu_mul_mx8(x[:, :32]),
                 lambda: uq_cuda.silu_mul_mx8(x, scales=torch.zeros(4, 2, dtype=torch.uint8, device="cuda")), lambda: uq_cuda.pack_fp4_weight(x[:, :40]), lambda: uq_cuda.pack_fp4_weight(x.double())):
        with pytest.raises(RuntimeError):
            call()


# -------------------------------------------------------------------------------------------------------------- linear
def _weight(N, K, seed, dtype=torch.float32):
    return uq_cuda.pack_fp4_weight(_rand((N, K), dtype, seed, K ** -0.5))


@gpu
@pytest.mark.parametrize("N,K,rule", [(1, 32, "ceil"), (200, 160, "ceil"), (256, 384, "paper")])
def test_pack_is_the_caches_encoder(N, K, rule):
    w = _rand((N, K), torch.bfloat16, 4)
    wc, ws = uq_cuda.pack_fp4_weight(w, rule=rule)
    ref = torch.nn.functional.pad(w, (0, -K % 128)).view(N, -1, 128)
    code, scale = torch.zeros(N, ref.shape[1], 1, 64, dtype=torch.uint8, device="cuda"), torch.zeros(N, ref.shape[1], 1, 4, dtype=torch.uint8, device="cuda")
    uq_cuda.quantize_on_write(ref, code, scale, torch.arange(N, device="cuda"), rule)
    rows = lambda t: t.transpose(1, 2).reshape(t.shape[0] * t.shape[2], -1)[:N]
    assert torch.equal(rows(wc), rows(code)) and torch.equal(rows(ws), rows(scale))
    assert (wc.transpose(1, 2).reshape(-1, wc.shape[1] * 64)[N:] == 0).all()


SHAPES = [(1, 128, 128), (1, 1, 32), (2, 130, 160), (3, 77, 736), (4, 500, 2048), (8, 256, 1024), (5, 1000, 1120), (17, 640, 4096), (33, 257, 96), (64, 384, 2048), (65, 129, 288), (127, 512, 256), (128, 300, 512), (130, 256, 640), (300, 128, 224)]


@gpu
@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_mx8_matches_the_plain_form(M, N, K, out):
    wc, ws = _weight(N, K, N)
    codes, scales, _ = uq_cuda.rms_norm_mx8(_rand((M, K), torch.float32, M))
    y = uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales, out_dtype=DT[out])
    assert y.shape == (M, N) and y.dtype == DT[out]
    check_linear(y, mx8_values(codes, scales), weight64(wc, ws, N, K), DT[out])


@gpu
@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_bf16_matches_the_plain_form(M, N, K, out):
    wc, ws = _weight(N, K, N + 1)
    x = _rand((M, K), torch.bfloat16, M)
    y = uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=DT[out])
    check_linear(y, _f64(x), weight64(wc, ws, N, K), DT[out], split=True)


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 8192), (3, 2048, 32768), (40, 20000, 1024), (16, 1024, 16384), (64, 19100, 416), (128, 20001, 288), (200, 9800, 160)])
def test_linear_long_and_wide(M, N, K):
    wc, ws = _weight(N, K, 5, torch.bfloat16)
    x = _rand((M, K), torch.bfloat16, 6)
    w64 = weight64(wc, ws, N, K)
    check_linear(uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32), _f64(x), w64, torch.float32, split=True)
    codes, scales, _ = uq_cuda.rms_norm_mx8(x)
    check_linear(uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales), mx8_values(codes, scales), w64, torch.bfloat16)


@gpu
def test_linear_many_rows_and_one():
    """More rows than any tile holds, and no row axis at all."""
    N, K = 384, 512
    wc, ws = _weight(N, K, 5)
    w64 = weight64(wc, ws, N, K)
    x = _rand((1000, K), torch.bfloat16, 6)
    check_linear(uq_cuda.fp4_linear(x, wc, ws, N), _f64(x), w64, torch.bfloat16, split=True)
    codes, scales, s = uq_cuda.rms_norm_mx8(x, None, x)
    check_linear(uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales), mx8_values(codes, scales), w64, torch.bfloat16)
    one, one_s, s1 = uq_cuda.rms_norm_mx8(x[7], None, x[7])
    assert one.shape == (K,) and one_s.shape == (K // 32,) and torch.equal(s1, s[7])
    assert torch.equal(one.view(torch.uint8), codes[7].view(torch.uint8)) and torch.equal(one_s, scales[7])
    y = uq_cuda.fp4_linear(one, wc, ws, N, scales=one_s, out_dtype=torch.float32)
    assert y.shape == (N,)
    check_linear(y[None], mx8_values(one, one_s)[None], w64, torch.float32)
    assert uq_cuda.fp4_linear(x[7], wc, ws).shape == (N,) and uq_cuda.silu_mul_mx8(x[7])[0].shape == (K // 2,)
    # rows that are not contiguous, codes and scales alike
    wide = torch.zeros(20, 2 * K, dtype=torch.uint8, device="cuda")
    wide[:, :K] = codes[:20].view(torch.uint8)
    wide_s = torch.zeros(K // 32, 20, dtype=torch.uint8, device="cuda")
    wide_s.copy_(scales[:20].t())
    got = uq_cuda.fp4_linear(wide[:, :K].view(torch.float8_e4m3fn), wc, ws, N, scales=wide_s.t())
    assert torch.equal(got, uq_cuda.fp4_linear(codes[:20].contiguous(), wc, ws, N, scales=scales[:20].contiguous()))


@gpu
def test_linear_every_code_and_scale():
    """All sixteen codes against all 256 e4m3 values, and scales over the whole range that products of fp32 hold."""
    wc = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(1, 1, 32, 1).view(1, 1, 128, 64).contiguous()
    ws = torch.full((1, 1, 128, 4), 127, dtype=torch.uint8, device="cuda")
    ws[0, 0, :, 0] = torch.arange(128, dtype=torch.uint8, device="cuda") + 60
    ws[0, 0, :, 2] = 200
    x = torch.zeros(254, 128, device="cuda")
    every = torch.tensor([b for b in range(256) if b & 127 != 127], dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    codes = x.to(torch.float8_e4m3fn)
    codes[:, 0] = every
    codes[:, 71] = every
    scales = torch.full((254, 4), 127, dtype=torch.uint8, device="cuda")
    scales[:, 0] = 100
    scales[:, 2] = torch.arange(254, dtype=torch.uint8, device="cuda") // 4 + 30
    y = uq_cuda.fp4_linear(codes, wc, ws, scales=scales, out_dtype=torch.float32)
    check_linear(y, mx8_values(codes, scales), weight64(wc, ws, 128, 128), torch.float32)


@gpu
@pytest.mark.parametrize("M", [7, 20, 40])
def test_linear_rows_do_not_touch_each_other_and_nothing_beyond_is_written(M):
    N, K = 200, 288
    wc, ws = _weight(N, K, 9)
    x = _rand((M, K), torch.bfloat16, 9)
    want = uq_cuda.fp4_linear(x, wc, ws, N)
    x[3, 7], x[5, 280], x[M - 1, 0] = float("nan"), float("inf"), float("-inf")
    buf = torch.full((M + 4, N), 5.0, dtype=torch.bfloat16, device="cuda")
    got = uq_cuda.fp4_linear(x, wc, ws, N, out=buf[2:M + 2])   # (2 * 200 * 2 bytes: on its 16-byte boundary)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[3, 5, M - 1]] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad]) and (buf[:2] == 5).all() and (buf[M + 2:] == 5).all()
    codes, scales, _ = uq_cuda.rms_norm_mx8(x)
    assert uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales)[3].isnan().all()
    # outputs that begin off a 16-byte boundary: rows of an odd width, and of a width that is a multiple of four
    for n, first in ((199, 1), (196, 3)):
        odd = torch.full((M + 4, n), 5.0, dtype=torch.bfloat16, device="cuda")
        wn, sn = _weight(n, K, 9)
        uq_cuda.fp4_linear(x, wn, sn, n, out=odd[first:M + first])
        assert torch.equal(odd[first:M + first][~bad], uq_cuda.fp4_linear(x, wn, sn, n)[~bad]) and (odd[:first] == 5).all() and (odd[M + first:] == 5).all()
    # zero rows and zero values
    assert uq_cuda.fp4_linear(x[:0], wc, ws, N).shape == (0, N)
    assert (uq_cuda.fp4_linear(torch.zeros(2, 3, K, dtype=torch.bfloat16, device="cuda"), wc, ws, N) == 0).all()


@gpu
def test_linear_small_and_large_values():
    """bf16 values at both ends of the type's range: their groups' scales reach the lower end of the byte (the weight is large, so
    that the products stay clear of fp32's subnormals)."""
    N, K = 128, 128
    wc, ws = _weight(N, K, 2)
    ws += 20
    x = _rand((4, K), torch.float32, 2)
    x = (x * torch.tensor([1e-36, 1e-39, 1e25, 1.0], device="cuda")[:, None]).bfloat16()
    w64 = weight64(wc, ws, N, K)
    y = uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32)
    x64 = _f64(x)
    want = x64 @ w64.T
    A = np.abs(x64) @ np.abs(w64).T
    # beside the usual: at a scale of 2^-127 a plane's last step is 2^-136
    assert (np.abs(_f64(y) - want) <= 2.0 ** -16 * A + 2.0 ** -135 * np.abs(w64).sum(1)).all()


@gpu
def test_linear_refuses_in_python():
    wc, ws = _weight(200, 288, 1)
    x = torch.zeros(4, 288, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: uq_cuda.fp4_linear(x.half(), wc, ws), lambda: uq_cuda.fp4_linear(x[:, :256], wc, ws), lambda: uq_cuda.fp4_linear(x, wc, ws, 300), lambda: uq_cuda.fp4_linear(x, wc, ws, 128),
                 lambda: uq_cuda.fp4_linear(x, wc, ws[:, :2].contiguous()), lambda: uq_cuda.fp4_linear(x, wc, ws, scales=torch.zeros(4, 9, dtype=torch.uint8, device="cuda")),
                 lambda: uq_cuda.fp4_linear(x, wc, ws, 200, out=torch.zeros(4, 256, device="cuda")), lambda: uq_cuda.fp4_linear(x, wc, ws, out_dtype=torch.float64),
                 lambda: uq_cuda.fp4_linear(x, wc, ws, 200, workspace=torch.zeros(10, device="cuda")),
                 lambda: uq_cuda.fp4_linear(x.repeat(3, 1), wc, ws, 200, workspace=torch.zeros(3000, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()


# -------------------------------------------------------------------------------------------- streams, graphs, a whole step
@gpu
def test_calls_on_another_stream_and_two_at_once():
    """Two streams at a time, each with its own inputs: what they give is what the default stream gave."""
    N, K = 640, 2048
    wc, ws = _weight(N, K, 1)
    xs = [_rand((24, K), torch.bfloat16, i) for i in range(2)]
    rs = [_rand((24, K), torch.bfloat16, 10 + i) for i in range(2)]

    def chain(x, r):
        codes, scales, s = uq_cuda.rms_norm_mx8(x, None, r)
        return uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales), uq_cuda.fp4_linear(s, wc, ws, N), *uq_cuda.silu_mul_mx8(torch.cat([s, x], 1))
    want = [chain(x, r) for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(chain(xs[i], rs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(g, want[i]))
    assert uq_cuda.last_status()[0] == 0


@gpu
def test_captured_and_replayed():
    """A step's operators in a CUDA graph, replayed on changed inputs, and two graphs whose calls share the caller's workspace on
    one stream."""
    N, K, M = 300, 1056, 9   # (nine bf16 rows: with the workspace)
    wc, ws = _weight(N, K, 1)
    x, r = _rand((M, K), torch.bfloat16, 1), _rand((M, K), torch.bfloat16, 2)
    work = torch.empty(uq_cuda.fp4_linear_scratch_bytes(M, K), dtype=torch.uint8, device="cuda")
    lens, starts = torch.tensor([40, 17], dtype=torch.int32, device="cuda"), torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda")
    table, free = torch.full((2, 4), 3, dtype=torch.int32, device="cuda"), torch.arange(20, 30, dtype=torch.int32, device="cuda")

    def step():
        codes, scales, s = uq_cuda.rms_norm_mx8(x, None, r)
        return (codes, scales, s, uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales), uq_cuda.fp4_linear(s, wc, ws, N, workspace=work),
                *uq_cuda.plan_step(lens, starts, table, 16, 12, free_pages=free))
    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (5, 6):
        x.copy_(_rand((M, K), torch.bfloat16, seed))
        lens.copy_(torch.tensor([33 + seed, 20], dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        want = step()
        for o in got:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(o, want))


@gpu
def test_the_same_bits_every_time():
    """Partial tiles are added in the order of their ranks, whichever CTA comes first."""
    for M, N, K in ((1, 4096, 4096), (33, 1000, 8192), (100, 512, 4096)):
        wc, ws = _weight(N, K, 3)
        x = _rand((M, K), torch.bfloat16, 4)
        want = uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32)
        for _ in range(20):
            assert torch.equal(uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32), want)


@gpu
@pytest.mark.parametrize("rotate,page", [(False, 64), (True, 16)])
def test_a_layers_step(rotate, page):
    """One layer of a verify step made of the operators and the attention they stand around: norm -> q, k, v -> slots and pages ->
    append -> verify -> output projection -> norm -> gate and up -> silu_mul -> down, against the same operators called one at
    a time on tables and slots worked out on the host; and the layer's output against 64 bits."""
    B, K, HQ, HKV, D, F = 3, 4, 8, 2, 128, 512
    H = HQ * D
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    w_qkv, w_o, w_gu, w_d = (uq_cuda.pack_fp4_weight(rnd(n, k) * k ** -0.5) for n, k in ((H + 2 * HKV * D, H), (H, H), (2 * F, H), (H, F)))
    lens0 = [37, 5, 130]
    pages = [-(-(n + K) // page) for n in lens0]
    held = [-(-n // page) for n in lens0]
    perm = torch.randperm(sum(pages) + 2, generator=g, device="cuda").to(torch.int32)
    width = max(pages) + 1
    bt = torch.full((B, width), 0, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        bt[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    free = perm[at:].contiguous()
    caches = [torch.zeros(len(perm), HKV, page, n, dtype=torch.uint8, device="cuda") for n in (D // 2, D // 32, D // 2, D // 32)]
    # what is stored already, through the operators as well: whole prompts
    lens_t = torch.tensor(lens0, dtype=torch.int32, device="cuda")
    slots0, taken0 = vllm_adapter.plan_step(lens_t, None, bt, page, sum(lens0))
    assert taken0 is None and (slots0 >= 0).all()
    vllm_adapter.append_kv(*caches, rnd(sum(lens0), HKV, D).bfloat16(), rnd(sum(lens0), HKV, D).bfloat16(), slots0, rotate_k=rotate)
    hidden, residual = rnd(B * K, H).bfloat16(), rnd(B * K, H).bfloat16()
    w1, w2 = (1 + 0.1 * rnd(H)).bfloat16(), (1 + 0.1 * rnd(H)).bfloat16()
    start = torch.arange(0, B * K + 1, K, dtype=torch.int32, device="cuda")
    assert vllm_adapter.eligible(hidden.view(-1, HQ, D), start, page) == (True, "ok", K)
    before = [t.clone() for t in caches]

    # the step, nothing between the calls that waits
    codes, scales, res = uq_cuda.rms_norm_mx8(hidden, w1, residual)
    qkv = uq_cuda.fp4_linear(codes, *w_qkv, scales=scales)
    slots, taken = vllm_adapter.plan_step(lens_t + K, start, bt, page, B * K, free_pages=free)
    k, v = qkv[:, H:H + HKV * D].reshape(-1, HKV, D), qkv[:, H + HKV * D:].reshape(-1, HKV, D)
    vllm_adapter.append_kv(*caches, k, v, slots, rotate_k=rotate)
    att = vllm_adapter.uq_verify_attention(qkv[:, :H].reshape(-1, HQ, D), *caches, bt, lens_t + K, K, rotate_q=rotate)
    o = uq_cuda.fp4_linear(att.view(-1, H), *w_o)
    codes2, scales2, res2 = uq_cuda.rms_norm_mx8(o, w2, res)
    gu = uq_cuda.fp4_linear(codes2, *w_gu, scales=scales2)
    c3, s3 = uq_cuda.silu_mul_mx8(gu)
    y = uq_cuda.fp4_linear(c3, *w_d, scales=s3)
    torch.cuda.synchronize()

    # tables and slots on the host
    want_bt, nxt, want_slots = bt.cpu().clone(), 0, []
    assert int(taken) == sum(pages) - sum(held)
    for b, n in enumerate(lens0):
        for j in range(held[b], pages[b]):
            assert want_bt[b, j] == free[nxt]
            nxt += 1
        want_slots += [int(want_bt[b, p // page]) * page + p % page for p in range(n, n + K)]
    assert slots.tolist() == want_slots
    # every link of the chain from its own inputs, in 64 bits
    s64 = _f64(hidden) + _f64(residual)
    check_mx8(codes, scales, s64 / np.sqrt((s64 ** 2).mean(-1, keepdims=True) + 1e-6) * _f64(w1))
    check_linear(qkv, mx8_values(codes, scales), weight64(*w_qkv, H + 2 * HKV * D, H), torch.bfloat16)
    ref = [t.clone() for t in before]
    uq_cuda.append_kv(*ref, k, v, torch.tensor(want_slots, device="cuda"), rotate_k=rotate)
    assert all(torch.equal(a, b) for a, b in zip(caches, ref))
    q4 = qkv[:, :H].reshape(B, K, HQ, D)
    assert torch.equal(att, uq_cuda.uq_decode_cuda(uq_cuda.fwht(q4) if rotate else q4, *ref, want_bt.cuda(), torch.tensor([n + K for n in lens0], device="cuda")).view_as(att))
    check_linear(o, _f64(att.view(-1, H)), weight64(*w_o, H, H), torch.bfloat16, split=True)
    s64 = _f64(o) + _f64(res)
    check_mx8(codes2, scales2, s64 / np.sqrt((s64 ** 2).mean(-1, keepdims=True) + 1e-6) * _f64(w2))
    check_linear(gu, mx8_values(codes2, scales2), weight64(*w_gu, 2 * F, H), torch.bfloat16)
    g64, u64 = _f64(gu)[:, :F], _f64(gu)[:, F:]
    check_mx8(c3, s3, g64 / (1 + np.exp(-g64)) * u64)
    check_linear(y, mx8_values(c3, s3), weight64(*w_d, H, F), torch.bfloat16)
    assert uq_cuda.last_status()[0] == 0


@gpu
def test_a_captured_step_follows_growing_requests():
    """The plan in a graph that is replayed as the requests grow: the lengths are the only input that changes, pages come from the
    free list's front, which the caller moves on by what was taken (a buffer's content, not its address)."""
    B, page, width, K = 5, 16, 40, 3
    table, lens = torch.full((B, width), -7, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    pool = torch.randperm(B * width, device="cuda").to(torch.int32)
    free = pool.clone()
    uq_cuda.plan_step(lens + 1, 1, table.clone(), page, B, free_pages=free)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lens += K
        slots, taken = uq_cuda.plan_step(lens, K, table, page, B * K + 2, free_pages=free)
        free.copy_(free[(torch.arange(len(pool), device="cuda") + taken) % len(pool)])
    n, used, want = 0, 0, np.full((B, width), -7, np.int32)
    host = pool.cpu().numpy()
    for _ in range(30):
        g.replay()
        want, want_slots, t = plan64([n + K] * B, [K] * B, want, page, B * K + 2, np.concatenate([host[used:], host[:used]]))
        n, used = n + K, used + t
        torch.cuda.synchronize()
        assert slots.tolist() == want_slots.tolist() and int(taken) == t and (table.cpu().numpy() == want).all()


@gpu
def test_ordinary_launches_give_the_same_bits(tmp_path):
    """UQ_B200_CFG=pdl=0 (read at a process's first launch): every launch an ordinary one."""
    import os
    import subprocess
    import sys
    from tests.conftest import ROOT
    code = """
import sys, torch
from all_quant_b200 import uq_cuda as U
g = torch.Generator(device="cuda").manual_seed(3)
x, r = (torch.randn(40, 1056, generator=g, device="cuda").bfloat16() for _ in range(2))
wc, ws = U.pack_fp4_weight(torch.randn(700, 1056, generator=g, device="cuda"))
c, s, t = U.rms_norm_mx8(x, None, r)
out = [c.view(torch.uint8), s, t, U.fp4_linear(c, wc, ws, 700, scales=s), U.fp4_linear(t, wc, ws, 700), U.fp4_linear(t[:3], wc, ws, 700), *(o.view(torch.uint8) for o in U.silu_mul_mx8(t[:, :1024]))]
bt = torch.full((2, 8), 5, dtype=torch.int32, device="cuda")
out += [*U.plan_step(torch.tensor([40, 17], dtype=torch.int32, device="cuda"), 9, bt, 16, 20, free_pages=torch.arange(9, dtype=torch.int32, device="cuda")), bt]
torch.save([o.cpu() for o in out], sys.argv[1])
"""
    results = []
    for cfg in ("", "pdl=0"):
        path = str(tmp_path / ("out" + cfg))
        subprocess.run([sys.executable, "-c", code, path], check=True, cwd=ROOT, env=dict(os.environ, UQ_B200_CFG=cfg), timeout=300)
        results.append(torch.load(path))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
@pytest.mark.parametrize("M,N,K,bf16", [(3, 256, 1024, True), (20, 256, 2048, False), (64, 300, 1024, True), (64, 19100, 256, True)])
def test_a_wait_that_runs_out_shows_in_the_output_and_the_next_call_is_right(M, N, K, bf16, monkeypatch):
    """The give-up path on a healthy GPU: with UQ_B200_CFG=expire=42 the first step's scales of x are never announced, so the issuing
    thread's wait for them - bounded at one second, like every wait - runs out.  The kernel returns (all roles drain, TMEM goes back), its
    outputs are NaN, the status record names a wait of these kernels, and the next call is right."""
    wc, ws = _weight(N, K, 8)
    x = _rand((M, K), torch.bfloat16, 8)
    codes, scales, _ = uq_cuda.rms_norm_mx8(x)
    call = (lambda: uq_cuda.fp4_linear(x, wc, ws, N)) if bf16 else (lambda: uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales))
    want = call()
    assert uq_cuda.last_status() == (0, 0, 0, 0) and not want.isnan().any()
    monkeypatch.setenv("UQ_B200_CFG", "expire=42")
    assert call().isnan().all()
    st = uq_cuda.last_status()
    assert st[0] == 1 and 40 <= st[2] < 60, st
    monkeypatch.delenv("UQ_B200_CFG")
    for _ in range(2):
        assert torch.equal(call(), want)
        assert uq_cuda.last_status() == (0, 0, 0, 0)


# ------------------------------------------------------------------------------------------------- edges of what is served
@gpu
def test_plan_around_the_default_size_of_shared_memory(tmp_path):
    """Three words of shared memory per request and the warps' sums: from B = 4085 on a launch has to ask for more than it gets unasked.  In a
    process of its own and in rising order, since a larger call raises the limit for those after it."""
    import subprocess
    import sys
    from tests.conftest import ROOT
    code = """
import numpy as np, torch
from all_quant_b200 import uq_cuda as U
for B in (4083, 4084, 4085, 4090, 4095, 4096, 16384):
    lens = np.random.default_rng(B).integers(1, 40, B)
    table, free = torch.full((B, 3), 5, dtype=torch.int32, device="cuda"), torch.arange(100, 100 + 3 * B, dtype=torch.int32, device="cuda")
    slots, taken = U.plan_step(torch.from_numpy(lens.astype(np.int32)).cuda(), 1, table, 16, B, free_pages=free)
    new, page = (lens - 1) % 16 == 0, np.full(B, 5)
    page[new] = 100 + np.arange(new.sum())
    assert int(taken) == new.sum() and (slots.cpu().numpy() == page * 16 + (lens - 1) % 16).all(), B
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, timeout=300)


def test_no_cta_of_the_products_ends_before_what_is_sent_to_it_or_issued_by_it():
    """The order that keeps a push from reaching a CTA that has ended, and a copy or an instruction from outliving its CTA, on the paths that give up too
    (read from the source: on a GPU the wrong order is a fault)."""
    from tests.test_kernel_order import kernels
    bodies = kernels("uq_linear.cu")
    body = bodies["uq_fp4_linear_kernel"]
    # behind the last barrier of a CTA in which anybody gave up: its pushes are waited for, with nothing that cuts the wait short
    assert body.rindex("__syncthreads();") < body.index("} else if (*abort_flag) {") < body.index("ended_wait(bar(C::oBarIn, 0), 0);")
    assert body.count("return;") == 1 and body.index("return;") < body.index("mbar_init")
    for body in bodies.values():
        # the copying threads see their copies land, the issuing thread its instructions end, whoever gave up
        assert body.rindex("bulk_load(") < body.rindex(", 51, j)" if ", 51, j)" in body else ", 41, j)") and "bounded_wait(" not in body.replace("if (!r) r = bounded_wait(", "")
        assert body.index("tc_commit(bar(C::oBarLast, 0));") < body.index("ended_wait(bar(C::oBarLast, 0), 0);") < body.index("tcgen05.dealloc")


@gpu
@pytest.mark.parametrize("M,N,K,bf16", [(3, 256, 1024, True), (8, 256, 1024, True), (20, 256, 2048, False), (64, 300, 1024, True)])
def test_one_cta_of_a_cluster_gives_up(M, N, K, bf16, monkeypatch):
    """UQ_B200_CFG=expire=43: only the last CTA of every cluster misses an arrival.  The others have pushed their partials long before it gives up, wait
    for its pushes, and stay until they have come: NaN everywhere, a record, and the next call is right."""
    wc, ws = _weight(N, K, 8)
    x = _rand((M, K), torch.bfloat16, 8)
    codes, scales, _ = uq_cuda.rms_norm_mx8(x)
    call = (lambda: uq_cuda.fp4_linear(x, wc, ws, N)) if bf16 else (lambda: uq_cuda.fp4_linear(codes, wc, ws, N, scales=scales))
    want = call()
    assert uq_cuda.last_status() == (0, 0, 0, 0) and not want.isnan().any()
    monkeypatch.setenv("UQ_B200_CFG", "expire=43")
    assert call().isnan().all()
    st = uq_cuda.last_status()
    assert st[0] == 1 and 40 <= st[2] < 60, st
    monkeypatch.delenv("UQ_B200_CFG")
    for _ in range(2):
        assert torch.equal(call(), want)
        assert uq_cuda.last_status() == (0, 0, 0, 0)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H", [64, 2048, 8192])
@pytest.mark.parametrize("eps", [2.0 ** -126, 2.0 ** -100, 2.0 ** -70, 1e-12])
def test_norm_of_tiny_rows(dtype, H, eps):
    """The smallest eps that is served and rows far below its root: a reciprocal root of up to 2^63, on values whose own products with a weight leave
    fp32's normal range.  (Nothing is added to the tolerance: a row is multiplied by powers of two only.)"""
    dt = DT[dtype]
    size = torch.tensor([2.0 ** -120, 2.0 ** -125, 2.0 ** -100, 2.0 ** -64, 2.0 ** -40, 2.0 ** -13, 0.0], device="cuda")
    x = (_rand((7, H), torch.float32, 3) * size[:, None]).to(dt)
    x[:, ::3] = 0
    x[2, 32:] *= 2.0 ** -20   # a group far above the others
    w = _rand((H,), torch.float32, 4)
    w[:32] *= 2.0 ** -24
    w = w.to(dt)
    x64, w64 = _f64(x), _f64(w)
    r = 1 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + float(np.float32(eps)))
    check_mx8(*uq_cuda.rms_norm_mx8(x, w, eps=eps)[:2], x64 * r * w64)
    check_mx8(*uq_cuda.rms_norm_mx8(x, eps=eps)[:2], x64 * r)
    codes, scales, s = uq_cuda.rms_norm_mx8(x, w, x, eps=eps)   # (the sum's doubling is exact, or zero)
    r = 1 / np.sqrt(((2 * x64) ** 2).mean(-1, keepdims=True) + float(np.float32(eps)))
    check_mx8(codes, scales, 2 * x64 * r * w64)
    assert (_f64(s) == 2 * x64).all()


def check_wide_range(y, x64, w64, dtype):
    """Products of bf16 rows whose groups span many binades: tighter than check_linear's `split`, whose bound is the group's largest value alone.
    What two planes leave out of a value is at most half a step of the second one, 2^-21 of the group's largest, and never more than the value.  It is let go
    where it is at most 2^-14 of the group's geometric mean (of the values that are not zero, by their bits); else two more planes hold it but for
    2^-21 of the largest that was left.  A wide group's channels are added in two steps more."""
    x = np.abs(x64).reshape(len(x64), -1, 32)
    bits = (x.astype(np.float32).view(np.uint32) >> 16).astype(np.int64)
    mean = ((bits.sum(2) // np.maximum((bits > 0).sum(2), 1)).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    left = np.minimum(x, 2.0 ** -21 * x.max(2, keepdims=True))
    lost = np.minimum(left, np.maximum(2.0 ** -14 * mean, 2.0 ** -21 * left.max(2))[..., None])
    A, K = np.abs(x64) @ np.abs(w64).T, x64.shape[1]
    y64 = x64 @ w64.T
    tol = (2 * K / 32 + 32) * 2.0 ** -22 * 1.125 * A + torch.finfo(dtype).eps / 2 * np.abs(y64) + lost.reshape(x64.shape) @ np.abs(w64).T
    assert (np.abs(y.double().cpu().numpy() - y64) <= tol).all()


def _wide_rows(M, K, every, ratio, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, 5::every] *= ratio
    return x.bfloat16()


@gpu
@pytest.mark.parametrize("every,ratio", [(1 << 20, 1e5), (32, 1e3), (32, 16384.0), (8, 1e5), (4, 1e3), (32, 1e9), (512, 1e30)])
@pytest.mark.parametrize("M,N,K", [(1, 200, 1024), (3, 130, 2080), (4, 256, 4096), (5, 200, 2080), (8, 128, 4096), (9, 300, 96), (16, 256, 1056), (20, 130, 2048), (33, 257, 1120), (64, 300, 2048),
                                   (100, 128, 1024), (64, 19100, 416)])
def test_linear_of_rows_with_large_channels(M, N, K, every, ratio):
    """A channel far larger than the others of its 32 whose codes in the weight are zero: the others count as they would without it."""
    g = torch.Generator(device="cuda").manual_seed(N)
    w = torch.randn(N, K, generator=g, device="cuda") * K ** -0.5
    w[:, 5::every] = 0
    wc, ws = uq_cuda.pack_fp4_weight(w)
    x = _wide_rows(M, K, every, ratio, M)
    w64 = weight64(wc, ws, N, K)
    assert (w64[:, 5::every] == 0).all()
    check_wide_range(uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32), _f64(x), w64, torch.float32)
    check_wide_range(uq_cuda.fp4_linear(x, wc, ws, N), _f64(x), w64, torch.bfloat16)


@gpu
@pytest.mark.parametrize("M,N,K", [(4, 200, 2048), (6, 200, 2048), (16, 256, 1056), (24, 200, 2048), (50, 300, 2048), (64, 19100, 416)])
def test_wide_rows_leave_their_neighbours_alone_and_repeat(M, N, K):
    """A row's bits do not depend on whether the rows beside it are of wide range, and are the same every time."""
    wc, ws = _weight(N, K, 4)
    x = _rand((M, K), torch.bfloat16, 5)
    plain = uq_cuda.fp4_linear(x, wc, ws, N, out_dtype=torch.float32)
    mixed = x.clone()
    mixed[1::2] = _wide_rows(M, K, 32, 1e5, 6)[1::2]
    mixed[1, 7] = float("inf")
    want = uq_cuda.fp4_linear(mixed, wc, ws, N, out_dtype=torch.float32)
    assert torch.equal(want[::2], plain[::2]) and want[1].isnan().all() and not want[2:].isnan().any()
    for _ in range(10):
        assert torch.equal(uq_cuda.fp4_linear(mixed, wc, ws, N, out_dtype=torch.float32)[2:], want[2:])
    work = torch.full((uq_cuda.fp4_linear_scratch_bytes(M, K),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(uq_cuda.fp4_linear(mixed, wc, ws, N, out_dtype=torch.float32, workspace=work)[2:], want[2:])


@gpu
def test_linear_picks_single_channels_of_any_size():
    """A weight of one channel per row: y is that channel.  To 2^-7 of itself or what an ordinary group's typical magnitude allows, whatever lies beside it."""
    K = 256
    w = torch.zeros(K, K, device="cuda")
    w[torch.arange(K), torch.arange(K)] = 1
    wc, ws = uq_cuda.pack_fp4_weight(w)
    for M in (2, 7, 12, 30, 60):
        x = (torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(M), device="cuda") * torch.tensor([1e-20, 1.0, 1e4, 1e9], device="cuda").repeat(K // 4)).bfloat16()
        check_wide_range(uq_cuda.fp4_linear(x, wc, ws, out_dtype=torch.float32), _f64(x), weight64(wc, ws, K, K), torch.float32)


@gpu
def test_linear_of_more_steps_than_a_cta_has_marks():
    """1172 steps of a CTA: a mark stands for two of them."""
    M, N, K = 5, 128, 1200000
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(N, K, generator=g, device="cuda")
    w[:, 5::50000] = 0
    wc, ws = uq_cuda.pack_fp4_weight(w)
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, 5::50000] *= 1e6
    x = x.bfloat16()
    w64 = weight64(wc, ws, N, K)
    check_wide_range(uq_cuda.fp4_linear(x, wc, ws, out_dtype=torch.float32), _f64(x), w64, torch.float32)


@gpu
@pytest.mark.parametrize("M", [1, 4, 9, 40])
def test_linear_into_its_own_input(M):
    """out in x's memory: every CTA reads all of x, and none may find another's outputs there."""
    K = 4096
    wc, ws = _weight(K, K, 7)
    x = _wide_rows(M, K, 500, 1e5, M)
    want = uq_cuda.fp4_linear(x, wc, ws)
    for _ in range(5):
        mine = x.clone()
        assert uq_cuda.fp4_linear(mine, wc, ws, out=mine) is mine and torch.equal(mine, want)
        both = torch.cat([x.view(-1), x.view(-1)])   # one that begins in the middle of x
        assert torch.equal(uq_cuda.fp4_linear(both[:M * K].view(M, K), wc, ws, out=both[M * K // 2:M * K // 2 + M * K].view(M, K)), want)
    codes, scales, _ = uq_cuda.rms_norm_mx8(x)
    want = uq_cuda.fp4_linear(codes, wc, ws, scales=scales)
    buf = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    mine = buf.view(torch.uint8).view(-1)[:M * K].view(M, K).view(torch.float8_e4m3fn)
    mine.copy_(codes)
    assert torch.equal(uq_cuda.fp4_linear(mine, wc, ws, scales=scales, out=buf), want)
    s = buf.view(torch.uint8).view(-1)[M * K:M * K + M * K // 32].view(M, K // 32)
    s.copy_(scales)
    assert torch.equal(uq_cuda.fp4_linear(codes, wc, ws, scales=s, out=buf), want)


@gpu
def test_linear_into_its_own_input_with_more_tiles_than_the_device_holds():
    """The same where some CTAs start when others have long written theirs."""
    M, K = 2, 40960
    g = torch.Generator(device="cuda").manual_seed(1)
    wc = torch.randint(0, 256, (K // 128, K // 128, 128, 64), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.full((K // 128, K // 128, 128, 4), 120, dtype=torch.uint8, device="cuda")
    x = _rand((M, K), torch.bfloat16, 3)
    want = uq_cuda.fp4_linear(x, wc, ws)
    for _ in range(3):
        mine = x.clone()
        assert torch.equal(uq_cuda.fp4_linear(mine, wc, ws, out=mine), want)


@gpu
def test_row_operators_into_their_own_inputs():
    """Codes, scales or the sum in memory of an input, not the same elements: the input is read as it was."""
    R, H = 3000, 512
    x, r, w = _rand((R, H), torch.bfloat16, 1), _rand((R, H), torch.bfloat16, 2), _rand((H,), torch.bfloat16, 3)
    same = lambda a, b: all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))
    want = uq_cuda.rms_norm_mx8(x, w, r)
    for _ in range(3):
        for first in (0, 1):   # which input shares its memory
            args = [x, r]
            buf = torch.cat([args[first].view(-1), torch.zeros(8 * H, dtype=torch.bfloat16, device="cuda")])
            args[first] = buf[:R * H].view(R, H)
            assert same(uq_cuda.rms_norm_mx8(args[0], w, args[1], sum_out=buf[7 * H:(R + 7) * H].view(R, H)), want)
        mine = x.clone()
        codes = mine.view(torch.uint8).view(-1)[R * H:].view(R, H).view(torch.float8_e4m3fn)   # the rows' second half
        assert same(uq_cuda.rms_norm_mx8(mine, w, r, codes=codes), want)
        mine = x.clone()
        scales = mine.view(torch.uint8).view(-1)[-R * H // 32:].view(R, H // 32)
        assert same(uq_cuda.rms_norm_mx8(mine, w, r, scales=scales), want)
        mine = x.clone()
        codes = mine.view(torch.uint8).view(-1)[:R * H // 2].view(R, H // 2).view(torch.float8_e4m3fn)
        assert same(uq_cuda.silu_mul_mx8(mine, codes=codes), uq_cuda.silu_mul_mx8(x))
    weight = torch.cat([w, torch.zeros(R * H // 32, dtype=torch.bfloat16, device="cuda")])
    assert same(uq_cuda.rms_norm_mx8(x, weight[:H], r, scales=weight.view(torch.uint8)[:R * H // 32].view(R, H // 32)), want)


def test_no_wide_group_is_overlooked():
    """The products' rule for groups of wide range (what two planes leave out of a value is more than 2^-14 of the geometric mean) is only asked where a lane's
    eight leading codes are, as whole numbers, under 84 on average: in numpy, over groups made to come close - a few values at, around and far below
    the border where two planes begin to lose bits, zeros among them - no group that the rule calls wide is passed over."""
    rng = np.random.default_rng(1)
    bf16 = lambda x: ((np.asarray(x, np.float32).view(np.uint32) + 0x8000) & np.uint32(0xffff0000)).view(np.float32).astype(np.float64)
    wide_groups = 0
    for _ in range(20):
        N = 10000
        v, low = rng.standard_normal((N, 32)), np.arange(32) < rng.integers(0, 32, (N, 1))
        kind, top = rng.integers(0, 6, (N, 1)), np.abs(v).max(1, keepdims=True)
        size = 2.0 ** rng.uniform(-40, 2, (N, 1))
        v = np.select([(kind == 0) & low, (kind == 1) & low, (kind == 2) & low, (kind == 3) & low, kind == 3, (kind == 4) & low, kind == 5],
                      [v * size, v * 2.0 ** rng.uniform(-30, 0, (N, 32)), top * 2.0 ** -14 * rng.uniform(0.3, 1, (N, 32)), np.sign(v) * size * rng.uniform(0.5, 1, (N, 32)),
                       448 * rng.uniform(0.5, 1, (N, 32)), np.zeros_like(v), v ** 5], v)
        x = bf16(v)
        E = exponent(np.abs(x).max(1))[:, None]
        hi = e4m3(np.ldexp(x, -E))
        rest = x - np.ldexp(hi, E)
        E2 = exponent(np.abs(rest).max(1))[:, None]
        left = np.abs(rest - np.ldexp(e4m3(np.ldexp(rest, -E2)), E2)).max(1)
        bits = (np.abs(x).astype(np.float32).view(np.uint32) >> 16).astype(np.int64)
        mean = ((bits.sum(1) // np.maximum((bits > 0).sum(1), 1)).astype(np.uint32) << 16).view(np.float32)
        codes = torch.from_numpy(np.abs(hi)).to(torch.float8_e4m3fn).view(torch.uint8).numpy().astype(np.int64).reshape(N, 4, 8).sum(2)
        wide = left > 2.0 ** -14 * mean
        wide_groups += wide.sum()
        assert ((codes < 8 * 84).any(1) | ~wide).all()
    assert wide_groups > 20000
