"""Cases for the NVFP4 expert operators: what each is timed and compared on.

NVFP4: a value is code * scale * global_scale, with an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and the
negatives; two per byte, the even element in the low nibble), one E4M3 scale for 16 consecutive
elements of a row and one float32 global scale for a tensor (or for each expert of a weight tensor).
The quantiser is defined by its float32 steps, so that every implementation gives the same codes
where a quotient lies next to a border: a block's scale is amax / (6 * global_scale) rounded to
E4M3, and its codes are x * (1 / (scale * global_scale)) rounded to E2M1, each operation rounded to
float32 once and each rounding to the nearest, halves to even, saturating.

`run` computes each operator in plain float32 torch operations where `own` is false and calls the
framework's operators where it is true; `exact` computes the same outputs from the definitions in
64 bits.
"""
import math

import torch

own = False

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------


def listed():
    return [
        # quantise and dequantise: the hidden state of one decoded token
        dict(name="roundtrip one token", op="roundtrip", groups=1, rows=1, k=7168, dtype="bf16"),
        # an fp16 activation of odd row count and a width that is no multiple of 32 elements
        dict(name="roundtrip odd fp16", op="roundtrip", groups=1, rows=1531, k=2064, dtype="fp16"),
        # gate/up weights of 16 experts, quantised while a checkpoint is loaded
        dict(name="roundtrip expert weights", op="roundtrip", groups=16, rows=4096, k=7168, dtype="bf16"),
        # a decode batch sent to its experts
        dict(name="permute 16 tokens", op="permute", tokens=16, experts=256, topk=8, hidden=7168, dropped=0.0),
        # a prompt batch sent to its experts, some slots pruned by adaptive gating
        dict(name="permute 4096 tokens", op="permute", tokens=4096, experts=256, topk=8, hidden=7168, dropped=0.1),
        # down product of one token's eight experts
        dict(name="product one token", op="product", experts=8, rows=8, n=7168, k=2048, even=True),
        # few ragged experts, some without rows, widths that end inside a tile
        dict(name="product ragged", op="product", experts=13, rows=777, n=1056, k=1088, even=False),
        # gate/up product of a long prompt: bound by the tensor cores
        dict(name="product long prompt", op="product", experts=16, rows=16384, n=4096, k=7168, even=False),
        # gate/up, SwiGLU, requantisation and down product of a decode batch
        dict(name="experts decode", op="experts", experts=64, rows=128, hidden=7168, inter=2048, limit=0.0),
        # the same for a prompt on small clamped experts
        dict(name="experts small prompt", op="experts", experts=32, rows=6000, hidden=2048, inter=768, limit=10.0),
        # the whole routed layer for one decoded token
        dict(name="layer one token", op="layer", tokens=1, experts=64, topk=8, hidden=7168, inter=2048, n_group=8, topk_group=4),
        # the whole routed layer for a prompt batch, at the framework's main configuration
        dict(name="layer 4096 tokens", op="layer", tokens=4096, experts=256, topk=8, hidden=7168, inter=2048, n_group=8, topk_group=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["roundtrip", "permute", "product", "experts", "layer"])
    if op == "roundtrip":
        groups = _log(rng, 1, 16)
        return dict(op=op, groups=groups, rows=_log(rng, 1, 4096), k=16 * _log(rng, 1, 448),
                    dtype=rng.choice(["bf16", "fp16"]))
    if op == "permute":
        topk = rng.randint(1, 8)
        return dict(op=op, tokens=_log(rng, 1, 4096), experts=rng.choice([16, 60, 64, 128, 256]), topk=topk,
                    hidden=64 * _log(rng, 2, 112), dropped=rng.choice([0.0, 0.25]))
    if op == "product":
        return dict(op=op, experts=_log(rng, 1, 64), rows=_log(rng, 1, 8192), n=32 * _log(rng, 1, 128),
                    k=64 * _log(rng, 1, 112), even=rng.random() < 0.3)
    if op == "experts":
        return dict(op=op, experts=_log(rng, 1, 32), rows=_log(rng, 1, 8192), hidden=64 * _log(rng, 2, 112),
                    inter=64 * _log(rng, 1, 32), limit=rng.choice([0.0, 10.0]))
    groups = rng.choice([1, 4, 8])
    experts = 8 * rng.choice([2, 4, 8])
    topk = rng.randint(1, 8)
    return dict(op=op, tokens=_log(rng, 1, 2048), experts=experts, topk=topk, hidden=64 * _log(rng, 2, 112),
                inter=64 * _log(rng, 2, 32), n_group=groups, topk_group=max(1, groups // 2))


# ---- inputs ------------------------------------------------------------------------------------


def _tile(scales, parts):
    """[E, N, K/16] scales in the order in which the matrix instruction takes them: tiles of 128 rows
    and 4 scales, row r of a tile at byte 16 * (r % 32) + 4 * (r // 32); the rows in `parts` equal
    parts, each filled up to whole tiles with zeros."""
    e, n, s = scales.shape
    rows, tall, wide = n // parts, -(-(n // parts) // 128), -(-s // 4)
    full = torch.zeros(e, parts, tall * 128, wide * 4, dtype=torch.uint8, device=scales.device)
    full[:, :, :rows, :s] = scales.view(torch.uint8).view(e, parts, rows, s)
    full = full.view(e, parts, tall, 4, 32, wide, 4).permute(0, 1, 2, 5, 4, 3, 6)
    return full.reshape(e, parts * tall, wide, 512).contiguous().view(torch.float8_e4m3fn)


def _weights(gen, experts, n, k, parts):
    """Random weights quantised expert by expert: codes, scales, tiled scales, global scales."""
    codes = torch.empty(experts, n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(experts, n, k // 16, dtype=torch.float8_e4m3fn, device="cuda")
    glob = torch.empty(experts, dtype=torch.float32, device="cuda")
    for e in range(experts):
        w = (torch.randn(n, k, generator=gen, device="cuda") * 0.02).to(torch.bfloat16).float()
        glob[e] = w.abs().max() / (6.0 * 448.0)
        mag, neg, s = _quantise(w, glob[e])
        idx = torch.where(mag <= 2, 2 * mag, torch.where(mag <= 4, mag + 2, 7.0)) + 8.0 * neg
        idx = idx.to(torch.uint8)
        codes[e] = idx[:, 0::2] | (idx[:, 1::2] << 4)
        scales[e] = s.to(torch.float8_e4m3fn)
    return dict(codes=codes, scales=scales, tiled=_tile(scales, parts), glob=glob)


def _activations(gen, rows, k):
    x = torch.randn(rows, k, generator=gen, device="cuda").to(torch.bfloat16)
    glob = torch.full((1,), 0.011, device="cuda")
    mag, neg, s = _quantise(x.float(), glob)
    idx = torch.where(mag <= 2, 2 * mag, torch.where(mag <= 4, mag + 2, 7.0)) + 8.0 * neg
    idx = idx.to(torch.uint8)
    return dict(codes=idx[:, 0::2] | (idx[:, 1::2] << 4), scales=s.to(torch.float8_e4m3fn), glob=glob)


def _plan(counts):
    """Expert offsets for the operators, and the padded row index of the plain form."""
    rows, most, experts = int(counts.sum()), max(1, int(counts.max())), counts.numel()
    offsets = torch.zeros(experts + 1, dtype=torch.int64)
    offsets[1:] = counts.cumsum(0)
    at = offsets[:-1, None] + torch.arange(most)[None]
    pad = at.clamp(max=max(0, rows - 1))
    expert = torch.repeat_interleave(torch.arange(experts), counts)
    back = expert * most + torch.arange(rows) - offsets[:-1][expert]
    return dict(offsets=offsets.to(torch.int32).cuda(), pad=pad.cuda(), back=back.cuda(), most=most)


def _counts(case, cpu):
    e, rows = case["experts"], case["rows"]
    if case.get("even", False):
        return torch.full((e,), rows // e, dtype=torch.int64) + (torch.arange(e) < rows % e)
    share = torch.rand(e, generator=cpu, dtype=torch.float64) + 0.25
    share[torch.rand(e, generator=cpu) < 0.1] = 0
    share[int(torch.randint(e, (1,), generator=cpu))] += 0.5
    return torch.bincount(torch.multinomial(share, rows, replacement=True, generator=cpu), minlength=e)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    op, st = case["op"], dict(case=case)
    if op == "roundtrip":
        shape = (case["groups"], case["rows"], case["k"])
        x = torch.randn(shape, generator=gen, device="cuda")
        x *= torch.exp(torch.randn(shape[0], shape[1], 1, generator=gen, device="cuda"))  # rows of unlike size
        st["x"] = x.to(TYPES[case["dtype"]])
        st["glob"] = st["x"].float().abs().amax(dim=(1, 2)) / (6.0 * 448.0)
    elif op == "permute":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        st["x"] = torch.randn(t, case["hidden"], generator=gen, device="cuda").to(torch.bfloat16)
        idx = torch.rand(t, e, generator=gen, device="cuda").argsort(dim=1)[:, :k]
        gone = torch.rand(t, k, generator=gen, device="cuda") < case["dropped"]
        st["idx"] = torch.where(gone, -1, idx).to(torch.int32).contiguous()
        st["glob"] = torch.full((1,), 0.0125, device="cuda")
    elif op == "product":
        st["plan"] = _plan(_counts(case, cpu))
        st["a"] = _activations(gen, case["rows"], case["k"])
        st["w"] = _weights(gen, case["experts"], case["n"], case["k"], 1)
    elif op == "experts":
        st["plan"] = _plan(_counts(case, cpu))
        st["a"] = _activations(gen, case["rows"], case["hidden"])
        st["gu"] = _weights(gen, case["experts"], 2 * case["inter"], case["hidden"], 2)
        st["down"] = _weights(gen, case["experts"], case["hidden"], case["inter"], 1)
        st["mid"] = torch.full((1,), 0.0078, device="cuda")
    else:
        t, e = case["tokens"], case["experts"]
        st["x"] = torch.randn(t, case["hidden"], generator=gen, device="cuda").to(torch.bfloat16)
        st["logits"] = torch.randn(t, e, generator=gen, device="cuda")
        st["bias"] = torch.randn(e, generator=gen, device="cuda") * 0.01
        st["gu"] = _weights(gen, e, 2 * case["inter"], case["hidden"], 2)
        st["down"] = _weights(gen, e, case["hidden"], case["inter"], 1)
        st["glob"] = torch.full((1,), 0.011, device="cuda")
        st["mid"] = torch.full((1,), 0.0078, device="cuda")
        _, idx = _gate(st["logits"], st["bias"], case)
        st["most"] = int(torch.bincount(idx.reshape(-1), minlength=e).max())  # rows of the fullest expert
    return st


# ---- plain forms -------------------------------------------------------------------------------


def _quantise(x, glob):
    """float32 x [..., K] and a global scale that broadcasts against x's blocks -> magnitudes of the
    codes, signs, block scales as float32."""
    b = x.unflatten(-1, (-1, 16))
    glob = glob.reshape(glob.shape + (1,) * (b.dim() - 1 - glob.dim())) if glob.dim() else glob
    s = (b.abs().amax(-1) / (6.0 * glob)).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    step = s * glob
    inv = torch.where(step > 0, 1.0 / step, 0.0)
    y = b * inv[..., None]
    a = y.abs().clamp(max=6.0)
    grid = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    mag = torch.round(a / grid) * grid  # halves go to the even code
    return mag.flatten(-2), torch.signbit(x), s


def _values(mag, neg, s, glob):
    """float32 values of a quantised tensor."""
    b = torch.where(neg, -mag, mag).unflatten(-1, (-1, 16)) * s[..., None]
    return b.flatten(-2) * glob


def _decode(q):
    """float32 code * scale (without the global scale) of codes and scales."""
    lut = torch.tensor(E2M1, device=q["codes"].device)
    pairs = torch.stack([lut.repeat(16), lut.repeat_interleave(16)], dim=1)  # byte -> two values
    v = pairs[q["codes"].int()].flatten(-2).unflatten(-1, (-1, 16))
    v *= q["scales"].float()[..., None]
    return v.flatten(-2)


def _grouped(a, w, plan, glob):
    """bf16 product of the rows of each expert with its weights: a [rows, K], w [E, N, K] float32."""
    y = torch.bmm(a[plan["pad"]], w.transpose(1, 2)) * glob[:, None, None]
    return y.flatten(0, 1)[plan["back"]].to(torch.bfloat16)


def _swiglu(gu, limit):
    g, u = gu.float().chunk(2, dim=-1)
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return (g / (1 + torch.exp(-g)) * u).to(torch.bfloat16)


def _experts(a, aglob, gu, down, mid, plan, limit):
    h = _swiglu(_grouped(a, _decode(gu), plan, aglob * gu["glob"]), limit).float()
    mag, neg, s = _quantise(h, mid)
    return _grouped(_values(mag, neg, s, 1.0), _decode(down), plan, mid * down["glob"])


def _gate(logits, bias, case):
    """Grouped sigmoid top-k: weights and experts in order of descending biased score."""
    t, e = logits.shape
    n, keep, k = case["n_group"], case["topk_group"], case["topk"]
    score = torch.sigmoid(logits.double()).float()  # next to equal scores order the experts
    biased = score + bias
    if n > 1:
        two = biased.view(t, n, e // n).sort(dim=-1, descending=True, stable=True)[0][..., :2].sum(-1)
        kept = two.sort(dim=-1, descending=True, stable=True)[1][:, :keep]
        open_ = torch.zeros(t, n, device=logits.device).scatter(1, kept, 1.0).bool()
        biased = biased.masked_fill(~open_.repeat_interleave(e // n, dim=1), float("-inf"))
    idx = biased.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    w = score.gather(1, idx)
    return w * (2.5 / w.sum(-1, keepdim=True)), idx


def _route(idx, experts):
    """Stable order of the slots by expert: offsets, slot -> row, row -> slot."""
    flat = torch.where(idx < 0, experts, idx).reshape(-1)
    perm = flat.argsort(stable=True)
    s2d = torch.empty_like(perm).scatter(0, perm, torch.arange(perm.numel(), device=perm.device))
    bounds = torch.arange(experts + 1, device=flat.device)
    return torch.searchsorted(flat[perm], bounds), s2d, perm


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _run_own(state, case, op)
    if op == "roundtrip":
        mag, neg, s = _quantise(state["x"].float(), state["glob"][:, None])
        return _values(mag, neg, s, state["glob"][:, None, None]).to(torch.bfloat16), s.to(torch.float8_e4m3fn)
    if op == "permute":
        x = state["x"].float()
        off, s2d, perm = _route(state["idx"].long(), case["experts"])
        mag, neg, s = _quantise(x, state["glob"])
        row = perm // case["topk"]
        v = _values(mag, neg, s, state["glob"]).to(torch.bfloat16)
        return v[row], s.to(torch.float8_e4m3fn).view(torch.uint8)[row].view(torch.float8_e4m3fn), off.int(), s2d.int(), perm.int()
    if op == "product":
        return _grouped(_decode(state["a"]), _decode(state["w"]), state["plan"], state["a"]["glob"] * state["w"]["glob"])
    if op == "experts":
        return _experts(_decode(state["a"]), state["a"]["glob"], state["gu"], state["down"], state["mid"], state["plan"], case["limit"])
    w, idx = _gate(state["logits"], state["bias"], case)
    off, s2d, perm = _route(idx, case["experts"])
    mag, neg, s = _quantise(state["x"].float(), state["glob"])
    rows = perm.numel()
    at = off[:-1, None] + torch.arange(state["most"], device=off.device)[None]
    expert = idx.reshape(-1)[perm]
    plan = dict(pad=at.clamp(max=rows - 1), back=expert * state["most"] + torch.arange(rows, device=off.device) - off[expert])
    a = _values(mag, neg, s, 1.0)[perm // case["topk"]]
    y = _experts(a, state["glob"], state["gu"], state["down"], state["mid"], plan, 0.0)
    slots = y[s2d].float().view(case["tokens"], case["topk"], -1)
    return (slots * w[..., None]).sum(1).to(torch.bfloat16)


# ---- the framework's operators -----------------------------------------------------------------


def _run_own(state, case, op):
    import layerstormexpertkernels_b200 as P

    if op == "roundtrip":
        codes, scales = P.nvfp4_quantize(state["x"], state["glob"])
        return P.nvfp4_dequantize(codes, scales, state["glob"]), scales
    if op == "permute":
        codes, scales, off, s2d, perm = P.moe_permute_nvfp4(state["x"], state["idx"], case["experts"], state["glob"])
        return P.nvfp4_dequantize(codes, scales, state["glob"]), scales, off, s2d, perm
    if op == "product":
        a, w = state["a"], state["w"]
        return P.grouped_gemm_nvfp4(a["codes"], a["scales"], w["codes"], w["tiled"], state["plan"]["offsets"], a["glob"], w["glob"])
    if op == "experts":
        a, gu, down, off = state["a"], state["gu"], state["down"], state["plan"]["offsets"]
        h, hs = P.grouped_gemm_swiglu_nvfp4(a["codes"], a["scales"], gu["codes"], gu["tiled"], off, a["glob"], gu["glob"], state["mid"], swiglu_limit=case["limit"])
        return P.grouped_gemm_nvfp4(h, hs, down["codes"], down["tiled"], off, state["mid"], down["glob"])
    gu, down = state["gu"], state["down"]
    return P.moe_layer_forward_nvfp4(state["x"], state["logits"], state["bias"], gu["codes"], gu["tiled"], gu["glob"],
                                     down["codes"], down["tiled"], down["glob"], case["topk"], case["n_group"], case["topk_group"],
                                     2.5, True, hidden_global_scale=state["glob"], inter_global_scale=state["mid"])


# ---- bytes and operations that a pass cannot do without ----------------------------------------


def work(case):
    op = case["op"]
    if op == "roundtrip":
        n = case["groups"] * case["rows"] * case["k"]
        return {"bytes": 2 * n + 2 * n + n / 16, "flops": 4 * n}
    if op == "permute":
        n, slots = case["tokens"] * case["hidden"], case["tokens"] * case["topk"]
        return {"bytes": 2 * n + slots * (12 + case["hidden"] * (2 + 1 / 16)), "flops": 4 * n}
    if op == "product":
        e, r, n, k = min(case["experts"], case["rows"]), case["rows"], case["n"], case["k"]
        return {"bytes": (e * n + r) * k * 0.5625 + 2 * r * n, "flops": 2 * r * n * k}
    h, i = case["hidden"], case["inter"]
    r = case["rows"] if op == "experts" else case["tokens"] * case["topk"]
    e = min(case["experts"], r)
    weights, flops = e * 3 * h * i * 0.5625, 6 * r * h * i
    if op == "experts":
        return {"bytes": weights + r * h * (0.5625 + 2), "flops": flops}
    return {"bytes": weights + case["tokens"] * (4 * h + 4 * case["experts"]), "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_quantise(x, glob):
    """float64 x [rows, K] and a float64 global scale -> float64 code * scale, and the scales: the
    definition's steps, each in 64 bits and then rounded to 32 as the definition says."""
    e4m3 = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    codes = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)

    def single(v):
        return v.float().double()

    def nearest(v, grid):
        hi = torch.searchsorted(grid, v.contiguous()).clamp(max=grid.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        below, above = v - grid[lo], grid[hi] - v
        up = (above < below) | ((above == below) & (hi % 2 == 0))
        return grid[torch.where(up, hi, lo)]

    b = x.view(x.shape[0], -1, 16)
    s = nearest(single(b.abs().amax(-1) / single(6 * glob)).clamp(max=448.0), e4m3)
    step = single(s * glob)[..., None]
    inv = torch.where(step > 0, single(1 / torch.where(step > 0, step, 1.0)), 0.0)
    y = single(b.abs() * inv).clamp(max=6.0)
    return (torch.copysign(nearest(y, codes), b) * s[..., None]).view(x.shape), s


def _exact_weights(q, e):
    c = q["codes"][e]
    lut = torch.tensor(E2M1, dtype=torch.float64, device=c.device)
    both = torch.stack([lut[(c & 15).long()], lut[(c >> 4).long()]], dim=-1).flatten(-2)
    return both * torch.repeat_interleave(q["scales"][e].double(), 16, dim=-1) * q["glob"][e].double()


def _round(x):
    return x.to(torch.bfloat16).double()


def _exact_ffn(a, gu, down, e, mid, limit):
    g, u = _round(a @ _exact_weights(gu, e).T).chunk(2, dim=-1)
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    h = _round(g * torch.sigmoid(g) * u)
    return (_exact_quantise(h, mid)[0] * mid) @ _exact_weights(down, e).T


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "roundtrip":
        vals = torch.empty(st["x"].shape, dtype=torch.float64, device="cuda")
        scales = torch.empty(st["x"].shape[:2] + (case["k"] // 16,), dtype=torch.float64, device="cuda")
        for i in range(case["groups"]):
            g = st["glob"][i].double()
            v, scales[i] = _exact_quantise(st["x"][i].double(), g)
            vals[i] = v * g
        return vals, scales
    if op == "permute":
        g = st["glob"].double()
        v, s = _exact_quantise(st["x"].double(), g)
        slot = st["idx"].long().reshape(-1)
        order = torch.sort(torch.where(slot < 0, case["experts"], slot), stable=True)[1]
        token = torch.div(order, case["topk"], rounding_mode="floor")
        return (v * g)[token], s[token], None, None, None
    if op == "layer":
        sig = 1 / (1 + torch.exp(-st["logits"].double()))
        pick = sig.float() + st["bias"]
        t, e, n = case["tokens"], case["experts"], case["n_group"]
        if n > 1:
            best = torch.topk(pick.view(t, n, -1), 2, dim=-1)[0].sum(-1)
            floor = torch.topk(best, case["topk_group"], dim=-1)[0][:, -1:]
            pick = torch.where((best >= floor).repeat_interleave(e // n, dim=1), pick, -torch.inf)
        chosen = torch.topk(pick, case["topk"], dim=-1)[1]
        w = sig.gather(1, chosen)
        w = 2.5 * w / w.sum(-1, keepdim=True)
        g, mid = st["glob"].double(), st["mid"].double()
        a = _exact_quantise(st["x"].double(), g)[0] * g
        out = torch.zeros_like(a)
        for i in range(e):
            token, slot = torch.nonzero(chosen == i, as_tuple=True)
            if token.numel():
                out.index_add_(0, token, w[token, slot][:, None] * _round(_exact_ffn(a[token], st["gu"], st["down"], i, mid, 0.0)))
        return out
    off = st["plan"]["offsets"].tolist()
    a = _exact_weights({k: v[None] for k, v in st["a"].items()}, 0)
    wide = case["n"] if op == "product" else case["hidden"]
    out = torch.empty(case["rows"], wide, dtype=torch.float64, device="cuda")
    for i in range(case["experts"]):
        lo, hi = off[i], off[i + 1]
        if hi > lo and op == "product":
            out[lo:hi] = a[lo:hi] @ _exact_weights(st["w"], i).T
        elif hi > lo:
            out[lo:hi] = _exact_ffn(a[lo:hi], st["gu"], st["down"], i, st["mid"].double(), case["limit"])
    return out
