"""The NVFP4 operators' refusals and host-side layout, without a GPU: the C
ABI rejects bad arguments before any CUDA call, the binding rejects tensors by
type, place and shape, and nvfp4_tile_scales puts every scale at its place."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import layerstormexpertkernels_b200 as P
from oracle import quant_oracle as Q

BAD, UNSUPPORTED = 1, 2
d = ctypes.c_void_p(256)      # never dereferenced: validation fails first
odd = ctypes.c_void_p(260)
z = ctypes.c_size_t(0)
i64 = ctypes.c_int64


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(P.LIBRARY_PATH)
    lib.lsek_last_error.restype = ctypes.c_char_p
    lib.lsek_moe_layer_nvfp4_workspace_size.restype = ctypes.c_size_t
    return lib


def test_quantize_refusals(lib):
    f = lib.lsek_nvfp4_quantize
    assert f(d, d, d, None, i64(1), i64(4), 24, 0, None) == BAD and b"multiple of 16" in lib.lsek_last_error()
    assert f(d, d, d, None, i64(1), i64(-1), 32, 0, None) == BAD
    assert f(d, d, d, None, i64(1), i64(4), 32, 2, None) == BAD      # fp32 input
    assert f(None, d, d, None, i64(1), i64(4), 32, 0, None) == BAD
    assert f(odd, d, d, None, i64(1), i64(4), 32, 0, None) == BAD    # codes on 8 bytes
    assert f(d, d, d, None, i64(1 << 30), i64(1 << 30), 32, 0, None) == BAD
    assert f(None, None, None, None, i64(1), i64(0), 32, 0, None) == 0
    g = lib.lsek_nvfp4_dequantize
    assert g(d, d, d, None, i64(1), i64(4), 8, 0, None) == BAD
    assert g(d, d, d, None, i64(1), i64(4), 32, 3, None) == BAD
    assert g(ctypes.c_void_p(264), d, d, None, i64(1), i64(4), 32, 0, None) == BAD  # out on 16 bytes
    assert g(None, None, None, None, i64(0), i64(4), 32, 0, None) == 0


def test_permute_refusals(lib):
    f = lib.lsek_moe_permute_nvfp4
    assert f(d, d, d, d, d, d, d, None, 4, 8, 40, 16, None) == BAD   # hidden % 16
    assert f(d, d, d, d, d, d, d, None, 4, 33, 64, 16, None) == BAD
    assert f(d, d, d, d, d, d, d, None, 4, 8, 64, 2000, None) == UNSUPPORTED
    assert f(None, d, d, d, d, d, d, None, 4, 8, 64, 16, None) == BAD
    assert f(odd, d, d, d, d, d, d, None, 4, 8, 64, 16, None) == BAD


def test_product_refusals(lib):
    f = lib.lsek_grouped_gemm_nvfp4

    def call(D=d, A=d, sa=d, B=d, sb=d, off=d, E=4, rows=8, N=64, K=64, ws=None):
        return f(D, A, sa, B, sb, off, None, None, E, rows, N, K, ws, z, None)

    assert call(K=96) == BAD and b"multiple of 64" in lib.lsek_last_error()
    assert call(N=48) == BAD
    assert call(K=0) == BAD
    assert call(E=0) == BAD
    assert call(E=1025) == UNSUPPORTED
    assert call(rows=-1) == BAD
    assert call(E=1024, N=1 << 21) == BAD       # weight rows past int32
    for name in ("D", "A", "sa", "B", "sb"):
        assert call(**{name: None}) == BAD
        assert call(**{name: ctypes.c_void_p(258) if name == "sa" else odd}) == BAD
    assert call(off=None) == BAD
    assert call(ws=ctypes.c_void_p(257)) == BAD
    assert call(rows=0, D=None, A=None) == 0
    g = lib.lsek_grouped_gemm_swiglu_nvfp4

    def gate(hc=d, hs=d, E=4, rows=8, I=64, K=64, limit=0.0):
        return g(hc, hs, d, d, d, d, d, None, None, None, E, rows, I, K, ctypes.c_float(limit), None, z, None)

    assert gate(I=48) == BAD and gate(K=32) == BAD and gate(limit=-1.0) == BAD
    assert gate(hc=None) == BAD and gate(hs=odd) == BAD
    assert gate(I=1 << 30) == BAD
    assert gate(rows=0) == 0


def test_layer_refusals(lib):
    class Gating(ctypes.Structure):
        _fields_ = [("T", ctypes.c_int32), ("E", ctypes.c_int32), ("k", ctypes.c_int32),
                    ("ng", ctypes.c_int32), ("tg", ctypes.c_int32), ("rsf", ctypes.c_float),
                    ("renorm", ctypes.c_int32), ("sf", ctypes.c_int32)]

    def call(T=4, E=16, k=2, H=128, I=64, limit=0.0, ws=d, wsb=1 << 30, w=d):
        p = Gating(T, E, k, 1, 1, 2.5, 1, 0)
        return lib.lsek_moe_layer_forward_nvfp4(
            d, d, d, None, w, d, None, d, d, None, None, None, ctypes.byref(p), H, I,
            ctypes.c_float(limit), None, None, ws, ctypes.c_size_t(wsb), None, None)

    assert call(T=0) == 0
    assert call(H=96) == BAD and call(I=32) == BAD
    assert call(limit=-1.0) == BAD
    assert call(E=1024) == UNSUPPORTED
    assert call(k=0) == BAD and call(E=0) == BAD
    assert call(w=odd) == BAD and call(w=None) == BAD
    assert call(ws=None) == BAD and call(wsb=100) == BAD and call(ws=odd) == BAD
    size = lib.lsek_moe_layer_nvfp4_workspace_size
    assert size(-1, 64, 64, 8, 2) == 0
    # codes and scales of x and h and the bf16 rows of the down product
    assert size(4096, 7168, 2048, 256, 8) >= 32768 * (9216 * 9 // 16 + 2 * 7168)


def test_binding_rejects_cpu_tensors():
    u = torch.zeros(2, 64, dtype=torch.uint8)
    s = torch.zeros(2, 8).to(torch.float8_e4m3fn)
    for f in (lambda: P.nvfp4_quantize(torch.zeros(2, 32, dtype=torch.bfloat16)),
              lambda: P.nvfp4_dequantize(u, s),
              lambda: P.moe_permute_nvfp4(torch.zeros(2, 32, dtype=torch.bfloat16),
                                          torch.zeros(2, 1, dtype=torch.int32), 4),
              lambda: P.grouped_gemm_nvfp4(u, s, u[None], s[None], torch.zeros(2, dtype=torch.int32)),
              lambda: P.grouped_gemm_swiglu_nvfp4(u, s, u[None], s[None], torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            f()


@pytest.mark.parametrize("nvfp4", [False, True])
def test_workspace_of_a_captured_graph_outlives_its_growth(nvfp4):
    """A captured graph keeps writing to the workspace that it was captured
    with, so that one stays allocated when a larger call outgrows it; one that
    no capture used is let go."""
    import weakref

    u8, f8 = torch.uint8, torch.float8_e4m3fn
    if nvfp4:
        layer = P.MoELayerNVFP4(torch.zeros(4, 128, 64, dtype=u8), torch.zeros(4, 2, 2, 512).to(f8), None,
                                torch.zeros(4, 128, 32, dtype=u8), torch.zeros(4, 1, 1, 512).to(f8), None, topk=2)
    else:
        layer = P.MoELayer(torch.zeros(4, 128, 64, dtype=torch.bfloat16),
                           torch.zeros(4, 64, 64, dtype=torch.bfloat16), topk=2)
    layer._ensure_workspace(4)
    first = weakref.ref(layer.workspace)
    layer._ensure_workspace(40)
    assert first() is None and layer.workspace.numel() >= layer.workspace_bytes(40)
    layer._capturing = lambda: True
    layer._ensure_workspace(30)
    captured = weakref.ref(layer.workspace)
    layer._capturing = lambda: False
    layer._ensure_workspace(4000)
    later = weakref.ref(layer.workspace)
    assert captured() is not None and captured() is not layer.workspace
    layer._ensure_workspace(8000)
    assert captured() is not None and later() is None
    layer._capturing = lambda: True
    layer._ensure_workspace(9000)  # grown inside a capture
    inside = weakref.ref(layer.workspace)
    layer._capturing = lambda: False
    layer._ensure_workspace(10000)
    assert inside() is not None and captured() is not None
    del layer
    assert captured() is None and inside() is None


def test_tile_scales_places_every_scale():
    gen = torch.Generator().manual_seed(0)
    for e, n, s, parts in [(1, 32, 4, 1), (2, 300, 12, 1), (3, 320, 8, 2), (1, 256, 4, 2)]:
        raw = torch.randint(0, 127, (e, n, s), generator=gen, dtype=torch.uint8)
        t = P.nvfp4_tile_scales(raw.view(torch.float8_e4m3fn), parts).view(torch.uint8)
        rows = n // parts
        tall = (rows + 127) // 128
        assert t.shape == (e, parts * tall, s // 4, 512)
        seen = torch.zeros_like(t)
        for i in range(e):
            for r in range(n):
                part, q = divmod(r, rows)
                for c in range(s):
                    at = (i, part * tall + q // 128, c // 4, 16 * (q % 32) + 4 * (q % 128 // 32) + c % 4)
                    assert t[at] == raw[i, r, c]
                    seen[at] = 1
        assert (t[seen == 0] == 0).all()


def test_tile_scales_refusals():
    f8 = torch.float8_e4m3fn
    for bad in (torch.zeros(1, 4, 4), torch.zeros(4, 4).to(f8), torch.zeros(1, 4, 6).to(f8)):
        with pytest.raises(ValueError):
            P.nvfp4_tile_scales(bad)
    with pytest.raises(ValueError):
        P.nvfp4_tile_scales(torch.zeros(1, 5, 4).to(f8), 2)
    with pytest.raises(ValueError):
        P.nvfp4_quantize_weights(torch.zeros(4, 64, dtype=torch.bfloat16))


def test_weight_global_scales():
    """The largest finite magnitude over 2688, 1 for zeros, at least 2^-100."""
    from layerstormexpertkernels_b200.nvfp4 import weight_global_scales
    w = torch.zeros(8, 4, 32, dtype=torch.bfloat16)
    w[0, 1, 5] = -3.0
    w[1, 2, 7], w[1, 0, 0] = 0.25, float("inf")
    w[2, 2, 7], w[2, 0, 0], w[2, 1, 1] = 0.25, float("nan"), -float("inf")
    w[3, 0, 0] = float("nan")
    w[4, 0, 3] = 2.0 ** -133   # the smallest bf16
    w[5, 0, 3] = 2.0 ** -95
    w[6, 3, 3] = torch.finfo(torch.bfloat16).max
    got = weight_global_scales(w).double()
    low = 2.0 ** -100
    want = torch.tensor([3 / 2688, 0.25 / 2688, 0.25 / 2688, 1.0, low, low,
                         torch.finfo(torch.bfloat16).max / 2688, 1.0], dtype=torch.float64)
    assert ((got - want).abs() <= want * 2.0 ** -24).all()
    assert w[1, 0, 0].isinf() and w[2, 0, 0].isnan()  # the weights stay as they are
    assert float(got[6]) < 2.0 ** 117
    assert weight_global_scales(w[:0]).shape == (0,) and (weight_global_scales(w[:, :0]) == 1).all()


def test_oracle_quantiser_is_nearest():
    """The oracle's codes against a search over all codes in 64 bits, away from
    the borders, and the ties on exact borders with a power-of-two scale."""
    gen = np.random.default_rng(0)
    y = gen.uniform(-7, 7, 4000).astype(np.float32)
    got = Q.E2M1_VALUES[Q.e2m1_encode(y)].astype(np.float64)
    best = np.abs(y[:, None].astype(np.float64) - Q.E2M1_VALUES[None]).min(1)
    assert np.array_equal(np.abs(got - y), best)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    assert Q.E2M1_VALUES[Q.e2m1_encode(ties)].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert Q.e2m1_encode(np.float32([-0.0, -0.1, -9.0])).tolist() == [8, 8, 15]
    packed, s = Q.nvfp4_quantize(np.float32([[0] * 16, [6] + [0] * 15, [1e30] + [0] * 15, [np.inf] * 16]), 1.0)
    assert s[:, 0].tolist() == [0, 0x38, 0x7E, 0x7F] and packed[:, 0].tolist() == [0, 7, 7, 0]
