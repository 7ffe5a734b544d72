"""GPU parity of the NVFP4 operators.

The quantiser, the dequantiser and the quantising permute are compared bit for
bit with the oracle.  The products are compared with 64-bit sums: an output is
off by its bf16 rounding (2^-8 of the value), the two fp32 multiplications
with the global scales, and the fp32 accumulation, for which each of the K/64
MMAs, and up to eight steps inside one, may lose 2^-23 of the sum of
magnitudes (`product_bound`).  The fused gate/up kernel and the layer are
compared bit for bit with the operators that they are made of."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from gpu_util import sync_and_check_device_error
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu


def pk():
    import layerstormexpertkernels_b200 as P
    return P


def u8(t: torch.Tensor) -> np.ndarray:
    return t.view(torch.uint8).cpu().numpy()


def glob(*v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def assert_same_codes(codes, scales, x: np.ndarray, g: float):
    want, want_s = Q.nvfp4_quantize(x, g)
    got, got_s = u8(codes).reshape(want.shape), u8(scales).reshape(want_s.shape)
    assert np.array_equal(got_s, want_s), f"{(got_s != want_s).sum()} scales differ"
    assert np.array_equal(got, want), f"{(got != want).sum()} bytes of codes differ"


def rand_fp4(gen, *shape):
    """Random codes and scales (any bits but the NaN scale), and their values."""
    k = shape[-1]
    codes = torch.randint(0, 256, shape[:-1] + (k // 2,), generator=gen, dtype=torch.uint8)
    s = torch.exp2(torch.randn(shape[:-1] + (k // 16,), generator=gen)).to(torch.float8_e4m3fn)
    vals = Q.nvfp4_values(codes.numpy().reshape(-1, k // 2), u8(s).reshape(-1, k // 16))
    return codes.cuda(), s.cuda(), vals.reshape(shape)


def product_bound(a, w, alpha):
    """(exact product, bound on |out - exact|) of float64 rows a and weights w."""
    exact, mag = alpha * (a @ w.T), alpha * (np.abs(a) @ np.abs(w).T)
    acc = (a.shape[1] / 64 + 8 + 2) * 2.0 ** -23 * mag
    return exact, acc + 2.0 ** -8 * (np.abs(exact) + acc)


def assert_product(out, a, w, offsets, alpha):
    got = out.float().cpu().numpy().astype(np.float64)
    for e in range(len(offsets) - 1):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            exact, bound = product_bound(a[lo:hi], w[e], alpha[e])
            over = np.abs(got[lo:hi] - exact) - bound
            assert over.max() <= 0, f"expert {e}: {over.max():.3e} over the bound"


# ---- quantise / dequantise --------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 7168), (3, 48), (257, 2064), (5, 64)])
@pytest.mark.parametrize("g", [1.0, 0.0125, 2.0 ** -9])
def test_quantize_equals_oracle(dtype, rows, k, g):
    gen = torch.Generator().manual_seed(rows * k)
    x = (torch.randn(rows, k, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))).to(dtype)
    codes, scales = pk().nvfp4_quantize(x.cuda(), glob(g))
    assert_same_codes(codes, scales, x.float().numpy(), g)
    if g == 1.0:
        again = pk().nvfp4_quantize(x.cuda())
        assert torch.equal(again[0], codes) and torch.equal(again[1].view(torch.uint8), scales.view(torch.uint8))


def test_quantize_every_bf16_value():
    """All 65536 bit patterns, one to a block that holds a value of one of six
    sizes beside it, so that each meets many quotients; infinities and NaNs
    among them give a NaN scale and codes of 0."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for other in (0.0, 1.0, 1.40625, 6.0, 0.0078125, 3000.0):
        x = torch.full((65536, 16), other, dtype=torch.bfloat16)
        x[:, 5] = bits
        x[:, 11] = 0.375 * other
        codes, scales = pk().nvfp4_quantize(x.cuda())
        assert_same_codes(codes, scales, x.float().numpy(), 1.0)


def test_quantize_borders_of_codes_and_scales():
    """Values that lie on and next to the borders of two codes for every E4M3
    scale, and amax values on the borders of two scales."""
    s = Q.e4m3_decode(np.arange(1, 127, dtype=np.uint8))
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=np.float32)
    x = np.zeros((s.size, 16), dtype=np.float32)
    x[:, :8] = s[:, None] * mid
    x[:, 8:15] = -x[:, :7]
    x[:, 15] = 6.0 * s
    edges = np.zeros((s.size - 1, 16), dtype=np.float32)
    edges[:, 3] = 6.0 * (s[:-1] + s[1:]) / 2
    for rows in (x, edges):
        for g in (1.0, 0.011, 1.0 / 3.0):
            t = torch.as_tensor(rows * np.float32(g)).to(torch.bfloat16)
            codes, scales = pk().nvfp4_quantize(t.cuda(), glob(g))
            assert_same_codes(codes, scales, t.float().numpy(), g)


def test_quantize_groups_and_unaligned_rows():
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(3, 7, 96, generator=gen).to(torch.bfloat16)
    g = [0.5, 0.01, 3.0]
    codes, scales = pk().nvfp4_quantize(x.cuda(), glob(*g))
    assert codes.shape == (3, 7, 48) and scales.shape == (3, 7, 6)
    for i in range(3):
        assert_same_codes(codes[i], scales[i], x[i].float().numpy(), g[i])
    flat = torch.zeros(1 + 7 * 96, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x[0].reshape(-1).cuda()
    odd = flat[1:].view(7, 96)  # starts 2 bytes past a 16-byte boundary
    assert odd.data_ptr() % 16 == 2
    codes, scales = pk().nvfp4_quantize(odd, glob(0.5))
    assert_same_codes(codes, scales, x[0].float().numpy(), 0.5)
    for shape in ((0, 32), (2, 0, 32), (4, 0)):
        c, s = pk().nvfp4_quantize(torch.empty(shape, dtype=torch.bfloat16, device="cuda"))
        assert c.numel() == 0 and s.numel() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequantize_every_code_and_scale(dtype):
    """All 256 code bytes with all 256 scale codes (negative scales and NaN
    included, as they may come in a file)."""
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(8).repeat(256, 1)  # [256, 2048]
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 256)
    for g in (1.0, 0.0007):
        got = pk().nvfp4_dequantize(codes.cuda(), scales.view(torch.float8_e4m3fn).cuda(), glob(g), dtype)
        assert got.dtype == dtype
        v = torch.as_tensor(Q.nvfp4_dequant(codes.numpy(), Q.e4m3_decode(scales.numpy())) * np.float32(g))
        want = v.to(dtype)
        same = (got.cpu() == want) | (got.cpu().isnan() & want.isnan())
        assert same.all()


def test_round_trip_is_near():
    """A block's values come back within half of the widest step of the codes
    (1 of 6, at the top) plus the rounding of the scale (2^-4)."""
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(64, 1024, generator=gen).to(torch.bfloat16).cuda()
    codes, scales = pk().nvfp4_quantize(x)
    back = pk().nvfp4_dequantize(codes, scales, dtype=torch.float32)
    amax = x.float().view(64, -1, 16).abs().amax(-1)
    err = (back - x.float()).view(64, -1, 16).abs().amax(-1)
    assert (err <= amax * (1 / 6 + 2.0 ** -4) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("exponent", [-131, -120, -105, -95, -60, 0, 60, 124])
def test_quantize_weights_of_any_size(exponent):
    """Weights from the smallest bf16 numbers to the largest come back within the
    codes' and scales' steps (of the block, and of the smallest scale, 2^-9, where
    the global scale is at its least), and a block with an infinity or a NaN is
    NaN alone."""
    P = pk()
    gen = torch.Generator().manual_seed(exponent + 200)
    w = torch.randn(3, 64, 256, generator=gen).clamp(-3.9, 3.9).to(torch.bfloat16)
    w = (w.double() * 2.0 ** exponent).to(torch.bfloat16).cuda()
    w[0, :, 32:48] = 0.0
    w[1, 5, 3], w[2, 7, 100], w[2, 9, 255] = float("inf"), float("nan"), -float("inf")
    codes, tiles, g = P.nvfp4_quantize_weights(w)
    rows = P.nvfp4_quantize(w, g)
    assert torch.equal(rows[0], codes)
    assert torch.equal(P.nvfp4_tile_scales(rows[1]).view(torch.uint8), tiles.view(torch.uint8))
    back = P.nvfp4_dequantize(codes, rows[1], g, torch.float32)
    blocks, got = w.double().view(3, 64, 16, 16), back.double().view(3, 64, 16, 16)
    amax = blocks.abs().amax(-1, keepdim=True)
    bad = ~amax.isfinite().expand_as(got)
    assert torch.equal(got.isnan(), bad) and int(bad.sum()) == 3 * 16
    # (1/6 of amax and 2^-4, float32's rounding of subnormal products: 2^-149)
    bound = amax * (1 / 6 + 2.0 ** -4) * (1 + 2.0 ** -20) + 6 * g.double().view(3, 1, 1, 1) * 2.0 ** -10 + 2.0 ** -149
    assert ((got - blocks).abs() <= bound)[~bad].all()


# ---- permute ----------------------------------------------------------------------


@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 16), (1, 8, 256, 7168), (37, 3, 11, 208), (300, 8, 64, 512),
                                     (5, 32, 40, 4112)])
def test_permute_quantizes_every_row(T, k, E, H):
    gen = torch.Generator().manual_seed(T + H)
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
    idx = torch.randint(0, E, (T, k), generator=gen, dtype=torch.int32)  # repeats allowed
    idx[torch.rand(T, k, generator=gen) < 0.2] = -1
    idx = idx.cuda()
    P = pk()
    codes, scales, off, s2d, perm = P.moe_permute_nvfp4(x, idx, E, glob(0.02))
    want = P.moe_permute(x, idx, E)
    for a, b in zip((off, s2d, perm), want[1:]):
        assert torch.equal(a, b)
    assert_same_codes(codes, scales, want[0].float().cpu().numpy(), 0.02)


def test_permute_empty_and_unaligned():
    P = pk()
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    out = P.moe_permute_nvfp4(x, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 8)
    assert out[0].shape == (0, 32) and out[2].tolist() == [0] * 9
    flat = torch.randn(1 + 6 * 48, device="cuda").to(torch.bfloat16)
    odd = flat[1:].view(6, 48)
    idx = torch.randint(0, 4, (6, 2), device="cuda", dtype=torch.int32)
    a, b = P.moe_permute_nvfp4(odd, idx, 4), P.moe_permute_nvfp4(odd.clone(), idx, 4)
    assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))


# ---- products ---------------------------------------------------------------------


def make_product(counts, n, k, seed, parts=1, pad_rows=0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(counts) + pad_rows
    a, asf, av = rand_fp4(gen, rows, k)
    w, wsf, wv = rand_fp4(gen, len(counts), n, k)
    off = [0] + list(np.cumsum(counts))
    tiles = pk().nvfp4_tile_scales(wsf, parts)
    return a, asf, av, w, tiles, wv, off, torch.tensor(off, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("counts,n,k", [
    ([1], 32, 64),
    ([16], 128, 64),
    ([17], 256, 256),
    ([32], 288, 320),
    ([33], 256, 512),
    ([128], 256, 256),
    ([129, 0, 1, 255, 193, 300], 256, 448),
    ([96, 97, 192, 200, 0, 0], 160, 1024),
    ([0, 5, 0, 31, 2], 7168, 2048),
    ([385, 40], 1056, 1088),
    ([40] * 16, 512, 7168),
])
def test_product_vs_64_bit_sum(counts, n, k):
    a, asf, av, w, tiles, wv, off, d_off = make_product(counts, n, k, seed=n + k + len(counts))
    gb = np.linspace(0.5, 2.0, len(counts)).astype(np.float32)
    out = pk().grouped_gemm_nvfp4(a, asf, w, tiles, d_off, glob(0.75), torch.as_tensor(gb).cuda())
    sync_and_check_device_error()
    assert_product(out, av, wv, off, 0.75 * gb.astype(np.float64))


@pytest.mark.parametrize("E,rows,n,k", [(8, 8192, 4096, 7168), (32, 6000, 2048, 768), (24, 7000, 3584, 2112)])
def test_product_of_many_units_a_block(E, rows, n, k):
    """Enough units that every block runs dozens of pipeline rounds at full load:
    each ring slot is refilled many times while its last readers are busy.  Three
    runs, each against the 64-bit sums, computed on the GPU."""
    P = pk()
    gen = torch.Generator(device="cuda").manual_seed(E)
    cpu = torch.Generator().manual_seed(E)
    counts = torch.bincount(torch.randint(0, E, (rows,), generator=cpu), minlength=E)
    off = torch.zeros(E + 1, dtype=torch.int32)
    off[1:] = counts.cumsum(0)
    x = torch.randn(rows, k, device="cuda", generator=gen).to(torch.bfloat16)
    w = (torch.randn(E, n, k, device="cuda", generator=gen) * 0.02).to(torch.bfloat16)
    ga = glob(0.011)
    a, asf = P.nvfp4_quantize(x, ga)
    wc, wt, gw = P.nvfp4_quantize_weights(w)
    av = P.nvfp4_dequantize(a, asf, None, torch.float32).double()  # code * scale, exact
    wv = P.nvfp4_dequantize(wc, P.nvfp4_quantize(w, gw)[1], None, torch.float32)
    outs = [P.grouped_gemm_nvfp4(a, asf, wc, wt, off.cuda(), ga, gw) for _ in range(3)]
    sync_and_check_device_error()
    for e in range(E):
        lo, hi = int(off[e]), int(off[e + 1])
        we, alpha = wv[e].double(), ga.double() * gw[e].double()
        exact, mag = alpha * (av[lo:hi] @ we.T), alpha * (av[lo:hi].abs() @ we.abs().T)
        acc = (k / 64 + 8 + 2) * 2.0 ** -23 * mag
        bound = acc + 2.0 ** -8 * (exact.abs() + acc)
        for out in outs:
            over = ((out[lo:hi].double() - exact).abs() - bound).max()
            assert over <= 0, f"expert {e}: {float(over):.3e} over the bound"


@pytest.mark.parametrize("rows", [1, 24, 100, 150, 230])
def test_product_exact_where_sums_are_exact(rows):
    """Scales that are powers of two: every partial sum is a multiple of 2^-6
    below 2^16, so fp32 sums are exact and each output is the bf16 rounding of
    the exact value, whatever the order."""
    gen = torch.Generator().manual_seed(rows)
    k, n = 256, 256
    codes_a = torch.randint(0, 256, (rows, k // 2), generator=gen, dtype=torch.uint8)
    codes_w = torch.randint(0, 256, (1, n, k // 2), generator=gen, dtype=torch.uint8)
    sa = torch.exp2(torch.randint(-2, 2, (rows, k // 16), generator=gen).float()).to(torch.float8_e4m3fn)
    sw = torch.exp2(torch.randint(-2, 2, (1, n, k // 16), generator=gen).float()).to(torch.float8_e4m3fn)
    av = Q.nvfp4_values(codes_a.numpy(), u8(sa))
    wv = Q.nvfp4_values(codes_w[0].numpy(), u8(sw[0]))
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    out = pk().grouped_gemm_nvfp4(codes_a.cuda(), sa.cuda(), codes_w.cuda(),
                                  pk().nvfp4_tile_scales(sw).cuda(), off)
    sync_and_check_device_error()
    want = torch.as_tensor((av @ wv.T).astype(np.float32)).to(torch.bfloat16)
    assert torch.equal(out.cpu(), want)


def test_each_scale_reaches_its_block():
    """One nonzero scale at a time: a product of ones sees exactly the block
    that the scale belongs to, for rows and columns on both sides of every
    32-row quarter and 128-row tile."""
    P = pk()
    k, n, rows = 512, 256, 160
    ones_a = torch.full((rows, k // 2), 0x22, dtype=torch.uint8, device="cuda")
    ones_w = torch.full((1, n, k // 2), 0x22, dtype=torch.uint8, device="cuda")
    sa = torch.zeros(rows, k // 16, device="cuda")
    sw = torch.zeros(1, n, k // 16, device="cuda")
    for r in range(rows):
        sa[r, r % (k // 16)] = 1 + r % 8
    sw[0] = torch.arange(k // 16, device="cuda") % 15 + 1
    sw[0, 1::2] = sw[0, 1::2].flip(-1)
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    f8 = torch.float8_e4m3fn
    out = P.grouped_gemm_nvfp4(ones_a, sa.to(f8), ones_w, P.nvfp4_tile_scales(sw.to(f8)), off)
    assert torch.equal(out.float(), 16 * (sa @ sw[0].T))
    sw.zero_()
    for c in range(n):
        sw[0, c, (5 * c) % (k // 16)] = 1 + c % 8
    sa[:] = torch.arange(k // 16, device="cuda") % 15 + 1
    out = P.grouped_gemm_nvfp4(ones_a, sa.to(f8), ones_w, P.nvfp4_tile_scales(sw.to(f8)), off)
    assert torch.equal(out.float(), 16 * (sa @ sw[0].T))
    sync_and_check_device_error()


def test_rows_of_an_expert_do_not_depend_on_their_neighbours():
    """A row's output has the same bits however many rows share its expert:
    alone, in a 32-row geometry, in one chunk or in several."""
    P = pk()
    a, asf, av, w, tiles, wv, off, d_off = make_product([430], 320, 1024, seed=3)
    full = P.grouped_gemm_nvfp4(a, asf, w, tiles, d_off)
    for rows in (1, 16, 31, 33, 95, 96, 97, 191, 192, 193, 385):
        part = P.grouped_gemm_nvfp4(a[:rows].contiguous(), asf[:rows].contiguous(), w, tiles,
                                    torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
        assert torch.equal(part, full[:rows]), rows
    sync_and_check_device_error()


def test_scales_that_start_at_a_4_byte_boundary():
    """A row of scales is a multiple of 4 bytes, and so is a slice's start."""
    P = pk()
    a, asf, av, w, tiles, wv, off, d_off = make_product([5, 200], 160, 512, seed=40)
    flat = torch.zeros(4 + asf.numel(), dtype=torch.uint8, device="cuda")
    flat[4:] = asf.view(torch.uint8).flatten()
    odd = flat[4:].view(torch.float8_e4m3fn).view(asf.shape)
    assert odd.data_ptr() % 16 == 4
    out = P.grouped_gemm_nvfp4(a, odd, w, tiles, d_off)
    assert torch.equal(out, P.grouped_gemm_nvfp4(a, asf, w, tiles, d_off))
    sync_and_check_device_error()


def test_rows_behind_the_last_expert_stay():
    """Rows outside every expert are not written (C ABI, canary output), with
    and without the workspace."""
    P = pk()
    a, asf, av, w, tiles, wv, off, d_off = make_product([30, 0, 200], 64, 128, seed=4, pad_rows=21)
    rows = a.shape[0]
    lib = ctypes.CDLL(P.LIBRARY_PATH)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for ws in (None, torch.full((256,), 255, dtype=torch.uint8, device="cuda")):
        d = torch.full((rows, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        st = lib.lsek_grouped_gemm_nvfp4(
            ptr(d), ptr(a), ptr(asf), ptr(w), ptr(tiles), ptr(d_off), None, None, 3, rows, 64, 128,
            ptr(ws) if ws is not None else None, ctypes.c_size_t(256 if ws is not None else 0),
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == 0
        sync_and_check_device_error()
        assert (d[230:] == 7.0).all()
        assert_product(d[:230], av, wv, off, [1.0] * 3)


@pytest.mark.parametrize("scratch", [0, 3, 4])
def test_many_units_without_a_counter(scratch):
    """The C ABI without scratch, and with less than a counter needs, shares units
    out by a fixed stride; with 4 bytes by the counter, whatever they hold: the
    bits of the binding's call, through both products.  The first expert starts
    behind 13 rows that belong to none and stay as they were, like those behind
    the last."""
    P = pk()
    counts, n, k = [300, 5, 0, 700, 190, 193, 60] * 5, 1024, 512
    a, asf, av, w, tiles, wv, off, _ = make_product(counts, n, k, seed=61, pad_rows=30)
    d_off = torch.tensor([o + 13 for o in off], dtype=torch.int32, device="cuda")
    rows, lo, hi = a.shape[0], 13, 13 + off[-1]
    lib = ctypes.CDLL(P.LIBRARY_PATH)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ws = torch.full((256,), 0xFF, dtype=torch.uint8, device="cuda")
    tail = (ptr(ws) if scratch else None, ctypes.c_size_t(scratch), stream)
    gate = P.nvfp4_tile_scales(rand_fp4(torch.Generator().manual_seed(62), len(counts), n, k)[1], 2)
    go = glob(8.0)
    d = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
    h = torch.full((rows, n // 4), 0xAB, dtype=torch.uint8, device="cuda")
    hs = torch.full((rows, n // 32), 0xAB, dtype=torch.uint8, device="cuda")
    assert lib.lsek_grouped_gemm_nvfp4(ptr(d), ptr(a), ptr(asf), ptr(w), ptr(tiles), ptr(d_off), None, None,
                                       len(counts), rows, n, k, *tail) == 0
    assert lib.lsek_grouped_gemm_swiglu_nvfp4(ptr(h), ptr(hs), ptr(a), ptr(asf), ptr(w), ptr(gate), ptr(d_off),
                                              None, None, ptr(go), len(counts), rows, n // 2, k,
                                              ctypes.c_float(0.0), *tail) == 0
    sync_and_check_device_error()
    want = P.grouped_gemm_nvfp4(a, asf, w, tiles, d_off)
    want_h, want_hs = P.grouped_gemm_swiglu_nvfp4(a, asf, w, gate, d_off, None, None, go)
    sync_and_check_device_error()
    for got, ref, old in ((d, want, 7.0), (h, want_h, 0xAB), (hs, want_hs.view(torch.uint8), 0xAB)):
        assert torch.equal(got[lo:hi], ref[lo:hi])
        assert (got[:lo] == old).all() and (got[hi:] == old).all()
    assert_product(d[lo:hi], av[lo:hi], wv, off, [1.0] * len(counts))


def test_products_captured_and_replayed():
    """A graph of gate/up and down product with more units than blocks: every
    replay zeroes its counters, and takes the inputs of the moment."""
    P = pk()
    counts, k = [300, 5, 0, 700, 190, 193, 60, 250], 1024
    gen = torch.Generator(device="cuda").manual_seed(71)
    x = torch.randn(sum(counts), k, generator=gen, device="cuda").to(torch.bfloat16)
    off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    gu, gut, gug = P.nvfp4_quantize_weights(torch.randn(8, 2 * 2048, k, generator=gen, device="cuda").to(torch.bfloat16), 2)
    dn, dnt, dng = P.nvfp4_quantize_weights(torch.randn(8, 5120, 2048, generator=gen, device="cuda").to(torch.bfloat16))
    ga, gh = glob(0.01), glob(300.0)

    def run():
        a, asf = P.nvfp4_quantize(x, ga)
        h, hs = P.grouped_gemm_swiglu_nvfp4(a, asf, gu, gut, off, ga, gug, gh)
        return h, hs, P.grouped_gemm_nvfp4(h, hs, dn, dnt, off, gh, dng)

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for rep in range(3):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        g.replay()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(got, run()))
    sync_and_check_device_error()


def test_nan_scale_reaches_only_its_row():
    """A block with a NaN scale (a non-finite activation) makes its token's
    outputs NaN and leaves the others as they were."""
    P = pk()
    x = torch.randn(50, 256, device="cuda").to(torch.bfloat16)
    clean, clean_s = P.nvfp4_quantize(x)
    x[17, 100] = float("inf")
    x[33, 3] = float("nan")
    codes, scales = P.nvfp4_quantize(x)
    gen = torch.Generator().manual_seed(1)
    w, wsf, _ = rand_fp4(gen, 1, 128, 256)
    off = torch.tensor([0, 50], dtype=torch.int32, device="cuda")
    tiles = P.nvfp4_tile_scales(wsf)
    out = P.grouped_gemm_nvfp4(codes, scales, w, tiles, off)
    want = P.grouped_gemm_nvfp4(clean, clean_s, w, tiles, off)
    sync_and_check_device_error()
    bad = torch.zeros(50, dtype=torch.bool, device="cuda")
    bad[[17, 33]] = True
    assert out[bad].isnan().all()
    assert torch.equal(out[~bad], want[~bad])


def test_product_without_rows_or_experts():
    P = pk()
    a, asf, av, w, tiles, wv, off, d_off = make_product([0, 0], 64, 128, seed=8)
    assert P.grouped_gemm_nvfp4(a, asf, w, tiles, d_off).shape == (0, 64)
    c, s = P.grouped_gemm_swiglu_nvfp4(a, asf, w, P.nvfp4_tile_scales(torch.zeros(2, 64, 8, device="cuda").to(torch.float8_e4m3fn), 2), d_off)
    assert c.shape == (0, 16) and s.shape == (0, 2)


@pytest.mark.parametrize("counts,inter,k,limit", [
    ([1], 32, 64, 0.0),
    ([20, 0, 7], 64, 256, 0.0),
    ([128, 5, 0, 200], 160, 256, 0.0),
    ([33, 193], 416, 1088, 10.0),
    ([64, 64], 256, 7168, 0.0),
    ([3, 0, 5, 1], 2048, 512, 1.5),
])
def test_swiglu_equals_product_swiglu_quantize(counts, inter, k, limit):
    P = pk()
    gen = torch.Generator().manual_seed(inter + k)
    x = torch.randn(sum(counts), k, generator=gen).to(torch.bfloat16).cuda()
    w = (torch.randn(len(counts), 2 * inter, k, generator=gen) * (2.0 / np.sqrt(k))).to(torch.bfloat16).cuda()
    off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    ga, go = glob(0.01), glob(0.02)
    a, asf = P.nvfp4_quantize(x, ga)
    wc, wt, gw = P.nvfp4_quantize_weights(w, 2)
    h, hs = P.grouped_gemm_swiglu_nvfp4(a, asf, wc, wt, off, ga, gw, go, swiglu_limit=limit)
    # the plain product takes the whole of [gate; up] as one part
    one = P.nvfp4_tile_scales(P.nvfp4_quantize(w, gw)[1], 1)
    gu = P.grouped_gemm_nvfp4(a, asf, wc, one, off, ga, gw)
    want, want_s = P.nvfp4_quantize(P.fused_swiglu(gu, swiglu_limit=limit), go)
    sync_and_check_device_error()
    assert torch.equal(hs.view(torch.uint8), want_s.view(torch.uint8))
    assert torch.equal(h, want)
    # and h against the formula in 64 bits from the bf16 g and u: fused_swiglu
    # is within a bf16 step (2^-7) of it, the quantiser within 1/6 + 2^-4 of amax
    g, u = gu.double().chunk(2, dim=-1)
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    exact = g * torch.sigmoid(g) * u
    back = P.nvfp4_dequantize(h, hs, go, torch.float32).double()
    amax = exact.abs().view(exact.shape[0], -1, 16).amax(-1)
    err = (back - exact).abs().view(exact.shape[0], -1, 16).amax(-1)
    smallest = 0.02 * 2.0 ** -10 * 6  # below this amax a scale rounds to 0
    assert (err <= amax * (1 / 6 + 2.0 ** -4 + 2.0 ** -7 + 1e-3) + smallest).all()


def same_as_three_operators(counts, inter, k, limit, seed, runs):
    """The fused kernel, `runs` times, against product + fused_swiglu + quantise."""
    P = pk()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(sum(counts), k, generator=gen, device="cuda").to(torch.bfloat16)
    w = (torch.randn(len(counts), 2 * inter, k, generator=gen, device="cuda") * (2.0 / np.sqrt(k))).to(torch.bfloat16)
    off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    ga, go = glob(0.01), glob(0.02)
    a, asf = P.nvfp4_quantize(x, ga)
    wc, wt, gw = P.nvfp4_quantize_weights(w, 2)
    got = [P.grouped_gemm_swiglu_nvfp4(a, asf, wc, wt, off, ga, gw, go, swiglu_limit=limit) for _ in range(runs)]
    one = P.nvfp4_tile_scales(P.nvfp4_quantize(w, gw)[1], 1)
    gu = P.grouped_gemm_nvfp4(a, asf, wc, one, off, ga, gw)
    want, want_s = P.nvfp4_quantize(P.fused_swiglu(gu, swiglu_limit=limit), go)
    sync_and_check_device_error()
    for h, hs in got:
        assert torch.equal(hs.view(torch.uint8), want_s.view(torch.uint8)) and torch.equal(h, want)
    return a, asf, w, gu, ga


@pytest.mark.parametrize("counts,inter,k,limit", [
    ([8] * 160, 160, 256, 0.0),                                            # one short unit after another
    ([95, 96, 97, 191, 192, 193, 0, 400, 1, 1000, 17, 33], 2048, 1088, 10.0),  # one and two accumulators, mixed
    ([700, 30, 811, 5, 640, 97] * 3, 1056, 2304, 0.0),
    ([1024, 300, 1500, 90, 2000, 64, 700, 1300], 2048, 7168, 0.0),         # full load
])
def test_swiglu_of_many_units_a_block(counts, inter, k, limit):
    """Several units for each block, so that accumulators, turning buffers and
    ring slots are used again: four runs with the bits of the three operators."""
    units = sum(-(-c // 192) for c in counts) * -(-inter // 128)
    assert units > 2 * 148
    a, asf, w, gu, ga = same_as_three_operators(counts, inter, k, limit, seed=len(counts) + k, runs=4)
    # and g, u against 64-bit sums, for the largest expert
    e = int(np.argmax(counts))
    lo = sum(counts[:e])
    P = pk()
    rows = P.nvfp4_dequantize(a[lo:lo + counts[e]], asf[lo:lo + counts[e]], None, torch.float32).double()
    we = w[e:e + 1].contiguous()
    wc, _, gw = P.nvfp4_quantize_weights(we, 2)
    wv = P.nvfp4_dequantize(wc, P.nvfp4_quantize(we, gw)[1], None, torch.float32)[0].double()
    alpha = ga.double() * gw.double()
    exact, mag = alpha * (rows @ wv.T), alpha * (rows.abs() @ wv.abs().T)
    acc = (k / 64 + 8 + 2) * 2.0 ** -23 * mag
    assert ((gu[lo:lo + counts[e]].double() - exact).abs() <= acc + 2.0 ** -8 * (exact.abs() + acc)).all()


def test_swiglu_of_more_than_256_experts():
    gen = torch.Generator().manual_seed(14)
    counts = [int(c) for c in torch.randint(0, 4, (300,), generator=gen)]
    counts[7], counts[299], counts[150] = 210, 97, 400
    same_as_three_operators(counts, 160, 320, 0.0, seed=15, runs=3)


def test_swiglu_for_every_gate_value():
    """Every bf16 gate magnitude and sign from 2^-126 up (128 significands as
    columns, 18 exponents and both signs as tokens, 15 experts for the rest of
    the exponents), with up values of the same exponent: the fused kernel's
    arithmetic gives the codes of fused_swiglu's."""
    P = pk()
    inter, k = 128, 256
    m = torch.arange(128, 256)
    w = torch.zeros(2 * inter, k // 16)  # element 0 of block i: bit i of the significand
    for i in range(8):
        w[:inter, i] = ((m >> i) & 1) * 2.0 ** i
    w[inter:, 8] = 128.0  # up row: 2^7, as the significand's top bit
    codes = torch.zeros(2 * inter, k // 2, dtype=torch.uint8)
    codes[:, ::8] = 2  # 1.0 at the first element of each block
    tokens = torch.zeros(36, k // 2, dtype=torch.uint8)
    tokens[:18, ::8], tokens[18:, ::8] = 2, 10
    ascale = torch.exp2(torch.arange(-9, 9).float()).repeat(2)[:, None].repeat(1, k // 16)
    E = 15
    off = torch.arange(E + 1, dtype=torch.int32, device="cuda") * 36
    gw = torch.exp2(torch.arange(E).float() * 18 - 124).cuda()
    a = tokens.repeat(E, 1).cuda()
    asf = ascale.repeat(E, 1).to(torch.float8_e4m3fn).cuda()
    wc = codes[None].repeat(E, 1, 1).cuda()
    wsf = w[None].repeat(E, 1, 1).to(torch.float8_e4m3fn).cuda()
    two, one = P.nvfp4_tile_scales(wsf, 2), P.nvfp4_tile_scales(wsf, 1)
    gu = P.grouped_gemm_nvfp4(a, asf, wc, one, off, None, gw)
    g = gu[:, :inter].float()
    finite = g[g.isfinite()]
    assert finite.abs().unique().numel() > 128 * 250  # the sweep is one
    for limit in (0.0, 10.0):
        h = P.fused_swiglu(gu, swiglu_limit=limit)
        for e in (-95, -60, -30, 0, 30, 60, 95):
            go = glob(2.0 ** e)
            got, got_s = P.grouped_gemm_swiglu_nvfp4(a, asf, wc, two, off, None, gw, go, swiglu_limit=limit)
            want, want_s = P.nvfp4_quantize(h, go)
            assert torch.equal(got_s.view(torch.uint8), want_s.view(torch.uint8))
            assert torch.equal(got, want)
    sync_and_check_device_error()


@pytest.mark.parametrize("limit", [0.0, 10.0])
def test_swiglu_has_every_bit_of_fused_swiglu(limit):
    """The fused kernel's h to the last bf16 bit, which its 4-bit outputs hide: a
    block has one value other than 0, so its scale is e4m3(|h| / (6 go)), and go
    goes through an eighth of an octave in steps of 0.35 %, finer than a bf16 step
    (0.39 % at least): for one of them a border of two scales lies between h and
    its neighbour.  (The same sweep with h one step up has to show it for every h
    of normal size.)  Gates: every bf16 magnitude from 2^-126 up and both signs;
    up values with other significands and with exponents of 9 below to 8 above
    the gate's range."""
    P = pk()
    inter, k, E = 2048, 256, 15
    b = torch.arange(128)
    w = torch.zeros(2 * inter, k // 16)  # rows 16 b: bit i of a significand at block i (gate) or 8 + i (up)
    for i in range(8):
        w[16 * b, i] = (((128 + b) >> i) & 1) * 2.0 ** i
        w[inter + 16 * b, 8 + i] = (((128 + 37 * b % 128) >> i) & 1) * 2.0 ** i
    codes = torch.zeros(2 * inter, k // 2, dtype=torch.uint8)
    codes[:, ::8] = 2  # 1.0 at the first element of each block
    signs, exps, ups = torch.tensor([2, 10]), torch.arange(-9, 9), torch.tensor([-9, 0, 8])
    n = len(signs) * len(exps) * len(ups)
    grid = torch.cartesian_prod(signs, exps, ups)
    tokens = torch.zeros(n, k // 2, dtype=torch.uint8)
    tokens[:, :64:8] = grid[:, :1].to(torch.uint8)
    tokens[:, 64::8] = 2
    ascale = torch.exp2(torch.cat([grid[:, 1:2].expand(n, 8), grid[:, 2:3].expand(n, 8)], 1).float())
    off = torch.arange(E + 1, dtype=torch.int32, device="cuda") * n
    gw = torch.exp2(torch.arange(E).float() * 18 - 124).cuda()
    a = tokens.repeat(E, 1).cuda()
    asf = ascale.repeat(E, 1).to(torch.float8_e4m3fn).cuda()
    wc = codes[None].repeat(E, 1, 1).cuda()
    wsf = w[None].repeat(E, 1, 1).to(torch.float8_e4m3fn).cuda()
    two, one = P.nvfp4_tile_scales(wsf, 2), P.nvfp4_tile_scales(wsf, 1)
    gu = P.grouped_gemm_nvfp4(a, asf, wc, one, off, None, gw)
    g = gu[:, :inter:16].float()
    assert g[g.isfinite()].abs().unique().numel() > 128 * 250
    h = P.fused_swiglu(gu, swiglu_limit=limit)
    # (2^128 is infinite in float32: the last expert's blocks are NaN)
    assert (h[:14 * n, 1::16] == 0).all()
    bits = h[:, ::16].contiguous().view(torch.int16)
    up = h.clone()
    up[:, ::16] = (bits + (bits & 0x7FFF < 0x7F7F).short()).view(torch.bfloat16)  # one step up, none past the largest
    shown = torch.zeros(g.shape, dtype=torch.bool, device="cuda")
    for e in range(-100, 101, 14):
        for i in range(36):
            go = glob(2.0 ** e * (1 + 0.0035 * i))
            got, got_s = P.grouped_gemm_swiglu_nvfp4(a, asf, wc, two, off, None, gw, go, swiglu_limit=limit)
            want, want_s = P.nvfp4_quantize(h, go)
            assert torch.equal(got_s.view(torch.uint8), want_s.view(torch.uint8)), (e, i)
            assert torch.equal(got, want), (e, i)
            shown |= P.nvfp4_quantize(up, go)[1].view(torch.uint8) != want_s.view(torch.uint8)
    size = h[:, ::16].float().abs()
    # within the scales' normal range of some go (2^-6 to 448, 6 go = 2^-97.4 to 2^96.6)
    normal = (size > 2.0 ** -103) & (size < 2.0 ** 105)
    normal[14 * n:] = False
    # by the formula in 64 bits 62908 of h without and 90864 with the clamp lie there
    assert normal.sum() > (90_000 if limit else 62_000) and shown[normal].all()
    sync_and_check_device_error()


def test_swiglu_clamp_keeps_nan():
    """A token with NaN among its values is NaN in every block behind the
    clamped gate/up kernel and behind the layer, and the other tokens are as
    without it; the plain product, fused_swiglu and the quantiser agree."""
    P = pk()
    layer, x, logits = make_layer(200, 8, 512, 192, 2, 1, 1, seed=17, limit=1.0)
    want = layer(x, logits)
    x[50, 7], x[120, 500], x[199, 0] = float("nan"), float("inf"), -float("inf")
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[50, 120, 199]] = True
    out = layer(x, logits)
    assert out[bad].isnan().all()
    assert not want.isnan().any() and torch.equal(out[~bad], want[~bad])
    w, idx = P.topk_gating(logits, layer.bias, 2, 1, 1, 2.5, True)
    a, asf, off, s2d, perm = P.moe_permute_nvfp4(x, idx, 8, layer.hidden_global_scale)
    args = (off, layer.hidden_global_scale, layer.w_gu_global_scale)
    h, hs = P.grouped_gemm_swiglu_nvfp4(a, asf, layer.w_gu, layer.w_gu_scales, *args,
                                        layer.inter_global_scale, swiglu_limit=1.0)
    rows = bad[perm.long() // 2]
    assert (hs.view(torch.uint8)[rows] == 0x7F).all() and (hs.view(torch.uint8)[~rows] != 0x7F).all()
    # the gate rows and the up rows apart, as the tiles hold them
    half = layer.w_gu.shape[1] // 2
    tall = layer.w_gu_scales.shape[1] // 2
    gu = torch.cat([P.grouped_gemm_nvfp4(a, asf, layer.w_gu[:, i * half:(i + 1) * half].contiguous(),
                                         layer.w_gu_scales[:, i * tall:(i + 1) * tall].contiguous(), *args)
                    for i in range(2)], 1)
    q, qs = P.nvfp4_quantize(P.fused_swiglu(gu, swiglu_limit=1.0), layer.inter_global_scale)
    assert torch.equal(q, h) and torch.equal(qs.view(torch.uint8), hs.view(torch.uint8))
    sync_and_check_device_error()


def test_more_than_256_experts():
    P = pk()
    gen = torch.Generator().manual_seed(12)
    counts = [int(c) for c in torch.randint(0, 4, (300,), generator=gen)]
    counts[7] = 210
    a, asf, av, w, tiles, wv, off, d_off = make_product(counts, 96, 128, seed=13)
    out = P.grouped_gemm_nvfp4(a, asf, w, tiles, d_off)
    sync_and_check_device_error()
    assert_product(out, av, wv, off, [1.0] * 300)


def test_no_expert_takes_a_row():
    """Rows but empty experts (every slot pruned): nothing is written."""
    P = pk()
    a, asf, av, w, tiles, wv, off, d_off = make_product([0, 0, 0], 64, 128, seed=2, pad_rows=40)
    lib = ctypes.CDLL(P.LIBRARY_PATH)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    d = torch.full((40, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    st = lib.lsek_grouped_gemm_nvfp4(ptr(d), ptr(a), ptr(asf), ptr(w), ptr(tiles), ptr(d_off), None, None,
                                     3, 40, 64, 128, None, ctypes.c_size_t(0),
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert st == 0
    sync_and_check_device_error()
    assert (d == 3.0).all()


def test_products_past_32_bits():
    """An output of more than 2^31 elements, and a quantised tensor of as many:
    the last rows are those of a small call on them alone."""
    P = pk()
    gen = torch.Generator().manual_seed(21)
    n, k, rows = 7168, 64, 300_000
    w, wsf, _ = rand_fp4(gen, 1, n, k)
    tiles = P.nvfp4_tile_scales(wsf)
    a = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda")
    asf = torch.ones(rows, k // 16, device="cuda").to(torch.float8_e4m3fn)
    out = P.grouped_gemm_nvfp4(a, asf, w, tiles, torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
    assert out.numel() > 2 ** 31
    small = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    for at in (0, 299_593 - 100, rows - 100):  # 299593 rows hold 2^31 elements
        want = P.grouped_gemm_nvfp4(a[at:at + 100].contiguous(), asf[at:at + 100].contiguous(), w, tiles, small)
        assert torch.equal(out[at:at + 100], want)
    codes, scales = P.nvfp4_quantize(out)
    back = P.nvfp4_dequantize(codes, scales)
    for at in (0, 299_593 - 100, rows - 100):
        c, s = P.nvfp4_quantize(out[at:at + 100].contiguous())
        assert torch.equal(codes[at:at + 100], c)
        assert torch.equal(back[at:at + 100], P.nvfp4_dequantize(c, s))
    sync_and_check_device_error()


def test_product_wider_than_2_31_elements_in_16_rows():
    """16 rows of 160 million columns: the rows of one 16-row chunk lie more than
    2^31 elements apart (14 * N > 2^31).  The whole output equals products with
    eight slices of the weights, each narrow enough for 32-bit offsets."""
    P = pk()
    n, k, rows, parts = 160_000_000, 64, 16, 8
    gen = torch.Generator(device="cuda").manual_seed(41)
    a = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    asf = torch.exp2(torch.randint(-2, 3, (rows, k // 16), device="cuda", generator=gen).float()).to(torch.float8_e4m3fn)
    w = torch.randint(0, 256, (1, n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    # n is a multiple of 128, so any bytes are tiles of scales: E4M3 codes of 0.25 to 1.875
    tiles = torch.randint(0x28, 0x40, (1, n // 128, k // 64, 512), dtype=torch.uint8, device="cuda",
                          generator=gen).view(torch.float8_e4m3fn)
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    out = P.grouped_gemm_nvfp4(a, asf, w, tiles, off)
    sync_and_check_device_error()
    step = n // parts
    assert step % 128 == 0 and 14 * n > 2 ** 31 and 16 * step < 2 ** 31
    for i in range(parts):
        part = P.grouped_gemm_nvfp4(a, asf, w[:, i * step:(i + 1) * step],
                                    tiles[:, i * step // 128:(i + 1) * step // 128], off)
        assert torch.equal(out[:, i * step:(i + 1) * step], part), i
    sync_and_check_device_error()


def test_product_with_2_gb_of_scales_a_tile():
    """K = 2^28 + 1024: a weight tile's scales take more than 2^31 bytes.  All
    codes but the last 2048 of a row are zeros, so the output is that of a
    product over the last 2048 alone."""
    P = pk()
    k, tail, n, rows = 2 ** 28 + 1024, 2048, 160, 3
    gen = torch.Generator(device="cuda").manual_seed(43)

    def ends(*shape):  # codes that are zeros but for the last `tail` of a row
        t = torch.zeros(*shape, k // 2, dtype=torch.uint8, device="cuda")
        t[..., -tail // 2:] = torch.randint(0, 256, (*shape, tail // 2), dtype=torch.uint8, device="cuda", generator=gen)
        return t

    a, w = ends(rows), ends(1, n)
    asf = torch.ones(rows, k // 16, device="cuda").to(torch.float8_e4m3fn)
    tiles = torch.full((1, 2, k // 64, 512), 0x38, dtype=torch.uint8, device="cuda")  # E4M3 1.0
    last = torch.randint(0x28, 0x40, (1, 2, tail // 64, 512), dtype=torch.uint8, device="cuda", generator=gen)
    tiles[:, :, -tail // 64:] = last
    f8 = torch.float8_e4m3fn
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    assert tiles[0, 0].numel() > 2 ** 31
    got = P.grouped_gemm_nvfp4(a, asf, w, tiles.view(f8), off)
    sync_and_check_device_error()
    want = P.grouped_gemm_nvfp4(a[:, -tail // 2:].contiguous(), asf[:, -tail // 16:].contiguous(),
                                w[:, :, -tail // 2:].contiguous(), last.view(f8), off)
    sync_and_check_device_error()
    assert want.abs().sum() > 0
    assert torch.equal(got, want)


def test_two_products_on_two_streams():
    """Two calls at once, each with its own stream and outputs, give what they
    give alone."""
    P = pk()
    cases = [make_product([400, 3, 250], 512, 1024, seed=31), make_product([30] * 40, 288, 576, seed=32)]
    want = [P.grouped_gemm_nvfp4(c[0], c[1], c[3], c[4], c[7]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(P.grouped_gemm_nvfp4(c[0], c[1], c[3], c[4], c[7]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    sync_and_check_device_error()


def test_refusals_on_the_gpu():
    """Types, shapes and places that the binding turns down before a launch."""
    P = pk()
    f8 = torch.float8_e4m3fn
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    codes, scales = P.nvfp4_quantize(x)
    bad_calls = [
        lambda: P.nvfp4_quantize(x.float()),
        lambda: P.nvfp4_quantize(x[:, :24].contiguous()),
        lambda: P.nvfp4_quantize(x.t()),
        lambda: P.nvfp4_quantize(x, torch.ones(2, device="cuda")),
        lambda: P.nvfp4_quantize(x, torch.ones(1)),
        lambda: P.nvfp4_quantize(x, torch.ones(1, dtype=torch.float64, device="cuda")),
        lambda: P.nvfp4_quantize(x[0]),
        lambda: P.nvfp4_dequantize(codes, scales[:, :2].contiguous()),
        lambda: P.nvfp4_dequantize(codes, scales.float()),
        lambda: P.nvfp4_dequantize(codes, scales, dtype=torch.float64),
        lambda: P.moe_permute_nvfp4(x.half(), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 4),
        lambda: P.moe_permute_nvfp4(x, torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 4),
        lambda: P.moe_permute_nvfp4(x, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 4),
        lambda: P.moe_permute_nvfp4(x, torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 1024),
    ]
    w = torch.zeros(2, 128, 32, dtype=torch.uint8, device="cuda")
    raw = torch.zeros(2, 128, 4, device="cuda").to(f8)
    tiles = P.nvfp4_tile_scales(raw)
    off = torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    ok = (codes, scales, w, tiles, off)

    def swap(i, t):
        return lambda: P.grouped_gemm_nvfp4(*(t if j == i else v for j, v in enumerate(ok)))

    bad_calls += [
        swap(0, codes[:, :16].contiguous()), swap(0, x), swap(1, scales.float()), swap(2, w[:, :, :16].contiguous()),
        swap(2, w[0]), swap(3, raw), swap(3, tiles[:1].contiguous()), swap(4, off[:2].contiguous()),
        swap(4, off.long()), swap(4, off.cpu()),
        lambda: P.grouped_gemm_nvfp4(*ok, torch.ones(2, device="cuda")),
        lambda: P.grouped_gemm_nvfp4(*ok, None, torch.ones(1, device="cuda")),
        lambda: P.grouped_gemm_swiglu_nvfp4(*ok),  # one part where two are due
    ]
    for i, call in enumerate(bad_calls):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            raise AssertionError(f"call {i} was taken")
    with pytest.raises(ValueError):  # swiglu_limit < 0, from the library
        P.grouped_gemm_swiglu_nvfp4(codes, scales, w, P.nvfp4_tile_scales(raw, 2), off, swiglu_limit=-1.0)
    assert P.grouped_gemm_nvfp4(*ok).shape == (4, 128)


@pytest.mark.parametrize("T,E,H,I,k,threshold", [(1, 8, 256, 64, 4, 0.5), (60, 16, 512, 128, 8, 0.6),
                                                 (300, 8, 320, 192, 2, 0.7)])
def test_chain_with_pruned_slots(T, E, H, I, k, threshold):
    """adaptive_gating -> moe_permute_nvfp4 -> gate/up -> down -> moe_unpermute,
    with NaN in every row behind the last expert that an operator leaves
    unwritten: a token is the sum over its kept slots (the first of a token is
    always kept; token T // 2 loses that one too)."""
    from oracle import moe_oracle as O
    from gpu_util import bits
    P = pk()
    gen = torch.Generator().manual_seed(T + E)
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
    w_gu = (torch.randn(E, 2 * I, H, generator=gen) / np.sqrt(H)).to(torch.bfloat16).cuda()
    w_down = (torch.randn(E, H, I, generator=gen) / np.sqrt(I)).to(torch.bfloat16).cuda()
    w, idx = P.topk_gating(torch.randn(T, E, generator=gen).cuda(), None, k, 1, 1, 2.5, True)
    w, idx, kept = P.adaptive_gating(w, idx, threshold)
    w[T // 2], idx[T // 2] = 0.0, -1
    valid = int((idx >= 0).sum())
    assert valid < T * k
    gx, gh = glob(0.01), glob(0.004)
    a, asf, off, s2d, _ = P.moe_permute_nvfp4(x, idx, E, gx)
    assert int(off[E]) == valid
    gu, gut, gug = P.nvfp4_quantize_weights(w_gu, 2)
    dn, dnt, dng = P.nvfp4_quantize_weights(w_down, 1)
    h, hs = P.grouped_gemm_swiglu_nvfp4(a, asf, gu, gut, off, gx, gug, gh)
    h[valid:] = 0xFF
    hs.view(torch.uint8)[valid:] = 0x7F  # NaN
    y = P.grouped_gemm_nvfp4(h, hs, dn, dnt, off, gh, dng)
    y[valid:] = float("nan")
    assert not y[:valid].isnan().any()
    out = P.moe_unpermute(y, w, s2d, T, k)
    sync_and_check_device_error()
    assert not out.isnan().any() and (out[T // 2] == 0).all()
    zeros = torch.where(torch.arange(T * k, device="cuda")[:, None] < valid, y, 0)
    assert np.array_equal(bits(out), O.moe_unpermute(bits(zeros), w.cpu().numpy(), s2d.cpu().numpy(), T, k))
    slots = (zeros.double()[s2d.long()].view(T, k, H) * w.double()[..., None])
    # k fp32 steps and one rounding to bf16
    bound = slots.abs().sum(1) * k * 2.0 ** -24 + slots.sum(1).abs() * 2.0 ** -8 * (1 + 2.0 ** -10)
    assert ((out.double() - slots.sum(1)).abs() <= bound).all()


# ---- the layer --------------------------------------------------------------------


def make_layer(T, E, H, I, k, n_group, topk_group, seed, limit=0.0):
    P = pk()
    gen = torch.Generator().manual_seed(seed)
    w_gu = (torch.randn(E, 2 * I, H, generator=gen) / np.sqrt(H)).to(torch.bfloat16).cuda()
    w_down = (torch.randn(E, H, I, generator=gen) / np.sqrt(I)).to(torch.bfloat16).cuda()
    bias = (torch.randn(E, generator=gen) * 0.01).cuda()
    layer = P.MoELayerNVFP4.from_weights(w_gu, w_down, bias, topk=k, n_group=n_group,
                                         topk_group=topk_group, swiglu_limit=limit,
                                         hidden_global_scale=glob(0.01), inter_global_scale=glob(0.004))
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
    logits = torch.randn(T, E, generator=gen).cuda()
    return layer, x, logits


def by_operators(layer, x, logits):
    """The layer's stages, one operator after the other."""
    P = pk()
    w, idx = P.topk_gating(logits, layer.bias, layer.topk, layer.n_group, layer.topk_group,
                           layer.routed_scaling_factor, layer.renormalize)
    a, asf, off, s2d, _ = P.moe_permute_nvfp4(x, idx, layer.num_experts, layer.hidden_global_scale)
    h, hs = P.grouped_gemm_swiglu_nvfp4(a, asf, layer.w_gu, layer.w_gu_scales, off,
                                        layer.hidden_global_scale, layer.w_gu_global_scale,
                                        layer.inter_global_scale, swiglu_limit=layer.swiglu_limit)
    y = P.grouped_gemm_nvfp4(h, hs, layer.w_down, layer.w_down_scales, off, layer.inter_global_scale,
                             layer.w_down_global_scale)
    return P.moe_unpermute(y, w, s2d, x.shape[0], layer.topk), w, idx


@pytest.mark.parametrize("T,E,H,I,k,ng,tg,limit", [
    (1, 16, 256, 128, 4, 4, 2, 0.0),
    (7, 8, 320, 192, 8, 1, 1, 0.0),
    (32, 16, 512, 64, 4, 4, 2, 10.0),
    (33, 16, 512, 256, 8, 8, 4, 0.0),
    (400, 8, 1024, 320, 2, 1, 1, 0.0),
])
def test_layer_equals_its_operators(T, E, H, I, k, ng, tg, limit):
    layer, x, logits = make_layer(T, E, H, I, k, ng, tg, seed=T + H, limit=limit)
    want, w, idx = by_operators(layer, x, logits)
    tw = torch.empty(T, k, device="cuda")
    ti = torch.empty(T, k, dtype=torch.int32, device="cuda")
    got = layer(x, logits, topk_weights=tw, topk_indices=ti)
    sync_and_check_device_error()
    assert torch.equal(ti, idx) and torch.equal(tw, w)
    assert torch.equal(got, want)
    P = pk()
    fn = P.moe_layer_forward_nvfp4(
        x, logits, layer.bias, layer.w_gu, layer.w_gu_scales, layer.w_gu_global_scale, layer.w_down,
        layer.w_down_scales, layer.w_down_global_scale, k, ng, tg, 2.5, True, swiglu_limit=limit,
        hidden_global_scale=layer.hidden_global_scale, inter_global_scale=layer.inter_global_scale,
        return_routing=True)
    assert torch.equal(fn[0], want) and torch.equal(fn[2], idx)


@pytest.mark.parametrize("T,E,H,I,k,ng,tg", [
    (300, 16, 2560, 2048, 4, 4, 2),
    (2100, 8, 2560, 2112, 2, 1, 1),
    (90, 320, 1536, 256, 8, 8, 4),      # more than 256 experts
    (1500, 320, 512, 128, 8, 1, 1),
])
def test_layer_of_many_units_on_a_dirty_workspace(T, E, H, I, k, ng, tg):
    """Both products have more units than blocks, so they share them out by the
    counters that the row copy zeroes: right on a workspace full of ones, on one
    that holds the counts of the call before, and at each replay of a graph."""
    units = [(T * k // 192 + min(E, T * k)) * n for n in (-(-I // 128), -(-H // 256))]
    assert min(units) > 148 and T * k > 192
    layer, x, logits = make_layer(T, E, H, I, k, ng, tg, seed=T + E)
    want = by_operators(layer, x, logits)[0]
    layer._ensure_workspace(T)
    layer.workspace.fill_(0xFF)
    assert torch.equal(layer(x, logits), want)
    assert torch.equal(layer(x, logits), want)
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(x, logits, out=out)
    for rep in range(3):
        if rep == 2:
            x.copy_(x.flip(0))
            want = by_operators(layer, x, logits)[0]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
    sync_and_check_device_error()


def test_layer_close_to_the_bf16_layer():
    """The 4-bit layer answers like the bf16 layer on the same weights.  A
    quantised operand is off by about 9.5 % rms: g and u by sqrt(2) of that
    (0.134), h = silu(g) u by about 0.134 * sqrt(1 + 1.2^2) = 0.21, the down
    product by sqrt(0.21^2 + 2 * 0.095^2) = 0.25, cos 1 / sqrt(1 + 0.25^2) =
    0.970; 0.95 allows an error of 0.33."""
    P = pk()
    gen = torch.Generator().manual_seed(2)
    E, H, I, T = 8, 1024, 512, 64
    w_gu = (torch.randn(E, 2 * I, H, generator=gen) / np.sqrt(H)).to(torch.bfloat16).cuda()
    w_down = (torch.randn(E, H, I, generator=gen) / np.sqrt(I)).to(torch.bfloat16).cuda()
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
    logits = torch.randn(T, E, generator=gen).cuda()
    kw = dict(topk=2, n_group=1, topk_group=1)
    got = P.MoELayerNVFP4.from_weights(w_gu, w_down, **kw)(x, logits).double().flatten()
    want = P.MoELayer(w_gu, w_down, **kw)(x, logits).double().flatten()
    cos = torch.dot(got, want) / (got.norm() * want.norm())
    assert cos > 0.95, float(cos)


def test_layer_captured_and_replayed_beside_another():
    """Two layers with workspaces of their own, captured on one stream each and
    replayed together on two streams, with inputs that change between replays."""
    cases = [make_layer(5, 16, 256, 128, 4, 4, 2, seed=1), make_layer(200, 8, 512, 192, 2, 1, 1, seed=2)]
    graphs = []
    for layer, x, logits in cases:
        out = torch.empty_like(x)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            layer(x, logits, out=out)  # grows the workspace before the capture
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            layer(x, logits, out=out)
        graphs.append((g, st, out))
    for rep in range(3):
        for (layer, x, logits), _ in zip(cases, graphs):
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(rep)).to(x.dtype))
        torch.cuda.synchronize()
        for g, st, _ in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (layer, x, logits), (_, _, out) in zip(cases, graphs):
            assert torch.equal(out, by_operators(layer, x, logits)[0])
    sync_and_check_device_error()


def test_layer_stage_events_and_empty_batch():
    P = pk()
    layer, x, logits = make_layer(40, 8, 256, 128, 2, 1, 1, seed=6)
    ev = P.StageEvents()
    layer(x, logits, stage_events=ev)
    torch.cuda.synchronize()
    assert set(ev.elapsed_ms()) == set(P.STAGES)
    assert layer(x[:0], logits[:0]).shape == (0, 256)


def test_replay_after_the_workspace_has_grown():
    """A graph captured for few tokens is replayed after an eager call of many
    has outgrown its workspace: the replay gives its bits and writes into no
    memory that was handed out since."""
    layer, x, logits = make_layer(500, 8, 512, 192, 2, 1, 1, seed=51)
    few, few_logits, out = x[:6].contiguous(), logits[:6].contiguous(), torch.empty_like(x[:6])
    layer(few, few_logits, out=out)
    size = layer.workspace.numel()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(few, few_logits, out=out)
    want = by_operators(layer, few, few_logits)[0]
    many = by_operators(layer, x, logits)[0]
    assert torch.equal(layer(x, logits), many) and layer.workspace.numel() > size
    taken = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(40)]
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all((t == 0x5A).all() for t in taken)
    assert torch.equal(layer(x, logits), many)
    sync_and_check_device_error()


def test_outgrown_workspace_waits_for_the_stream_that_uses_it():
    """A workspace that came from the default stream and is outgrown on another
    is handed out again only when that stream has done with it."""
    layer, x, logits = make_layer(500, 8, 512, 192, 2, 1, 1, seed=52)
    few, few_logits = x[:6].contiguous(), logits[:6].contiguous()
    want, many = layer(few, few_logits), by_operators(layer, x, logits)[0]
    old, size = layer.workspace.data_ptr(), layer.workspace.numel()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
        a = layer(few, few_logits)
        b = layer(x, logits)
    taken = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(40)]
    assert not st.query(), "the stream was done too early for the test to say anything"
    assert all(t.data_ptr() != old for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, many)
    sync_and_check_device_error()
