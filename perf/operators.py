"""Measured cases of the operators around a product: rotary positions with several axes, dropout from a counter-based
generator, and group norm with an activation over channels that lie last.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) where
``own`` is false, and through ``l2_torch_alloc_amd.ops`` where it is true.
"""
import functools
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------

def _rope(name, batch, tokens, q_heads, k_heads, head_dim, sections, dtype, half, order, backward, rows):
    return {"name": name, "op": "rope_axes", "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads,
            "head_dim": head_dim, "sections": ",".join(str(s) for s in sections), "dtype": dtype, "half": half,
            "order": order, "backward": backward, "rows": rows}


def _dropout(name, rows, width, p, dtype, residual, backward):
    return {"name": name, "op": "dropout", "rows": rows, "width": width, "p": p, "dtype": dtype, "residual": residual,
            "backward": backward}


def _norm(name, batch, pixels, channels, groups, activation, dtype, weights, backward):
    return {"name": name, "op": "group_norm", "batch": batch, "pixels": pixels, "channels": channels, "groups": groups,
            "activation": activation, "dtype": dtype, "weights": weights, "backward": backward}


def listed():
    return [
        # one new token for each of 16 requests, text behind images: all three axes, grouped-query heads; latency counts
        _rope("rope_axes_decode", 16, 1, 32, 8, 128, (16, 24, 24), "bf16", True, "blocks", False, 32768),
        # a training step over images and text: 4 sequences of 4096 tokens, grouped-query heads
        _rope("rope_axes_train", 4, 4096, 32, 8, 128, (16, 24, 24), "bf16", False, "blocks", False, 8192),
        # the gradient of a video's tokens (odd count), axes dealt in turn so that each sees all frequencies
        _rope("rope_axes_video_grad", 1, 13 * 33 * 45, 24, 24, 128, (24, 20, 20), "fp32", True, "turns", True, 1024),
        # patches of 8 images in an encoder: two axes, 16 heads of 64
        _rope("rope_axes_patches", 8, 1369, 16, 16, 64, (16, 16), "fp16", False, "blocks", False, 64),
        # a short batch of one small layer; latency counts
        _dropout("dropout_small", 7, 1031, 0.1, "bf16", False, False),
        # the end of a transformer layer in training: dropout of the branch, added to the residual
        _dropout("dropout_residual", 16384, 4096, 0.1, "bf16", True, False),
        # the gradient of such a layer; ragged rows of packed sequences
        _dropout("dropout_grad", 9973, 2561, 0.25, "fp16", False, True),
        # 32-bit activations, an odd count
        _dropout("dropout_fp32", 4099, 1027, 0.5, "fp32", False, False),
        # the innermost resolution of an image model: 2 images of 8x8; latency counts
        _norm("norm_inner", 2, 64, 1280, 32, "silu", "bf16", "fp32", False),
        # its outer resolution in training, forward: 10 channels in a group
        _norm("norm_outer", 8, 64 * 64, 320, 32, "silu", "bf16", "fp32", False),
        # the last stage of an image decoder: one image of 512x512
        _norm("norm_decoder", 1, 512 * 512, 256, 32, "silu", "fp16", "same", False),
        # a training step's gradient at the middle resolution
        _norm("norm_grad", 16, 32 * 32, 640, 32, "silu", "bf16", "fp32", True),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope_axes", "dropout", "group_norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    backward = rng.random() < 0.4
    if op == "rope_axes":
        half = rng.random() < 0.5
        head_dim = rng.choice([32, 64, 128, 256] if half else [32, 64, 72, 80, 96, 128, 256])
        pairs, axes = head_dim // 2, rng.choice([2, 3, 3])
        unit = rng.choice([1, 4])
        cuts = sorted(rng.sample(range(1, pairs // unit), axes - 1))
        ends = [0] + [c * unit for c in cuts] + [pairs]
        sections = [b - a for a, b in zip(ends, ends[1:])]
        k_heads = rng.choice([1, 2, 3, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 3, 4])
        batch = rng.choice([1, 2, 3, 8, 16])
        most = max(1, (1 << 26) // ((q_heads + k_heads) * head_dim * batch))
        tokens = rng.choice([1, _between(rng, 1, most), _between(rng, 1, most)])
        case = _rope("", batch, tokens, q_heads, k_heads, head_dim, sections, dtype, half, rng.choice(["blocks", "turns"]), backward,
                     rng.choice([64, 1000, 8192, 40961]))
    elif op == "dropout":
        width = rng.choice([_between(rng, 1, 8192), rng.choice([64, 512, 1024, 4096, 8192])])
        case = _dropout("", _between(rng, 1, max(1, (1 << 25) // width)), width, rng.choice([0.0, 0.05, 0.1, 0.3, 0.5, 0.9]), dtype,
                        (not backward) and rng.random() < 0.5, backward)
    else:
        groups = rng.choice([1, 4, 8, 16, 32, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 6, 8, 10, 16, 20, 40])
        batch = rng.choice([1, 2, 3, 8, 16])
        pixels = rng.choice([1, _between(rng, 1, max(1, (1 << 25) // (channels * batch))), _between(rng, 64, max(64, (1 << 25) // (channels * batch)))])
        if pixels * channels // groups < 8:        # a group of so few values has next to no spread to divide by
            pixels = 8
        case = _norm("", batch, pixels, channels, groups, rng.choice(["none", "silu", "silu"]), dtype, rng.choice(["fp32", "same"]), backward)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------

def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def _pair_axis(sections, order):
    """The axis of every pair of a head: section after section, or dealt to the axes in turn until each has its share."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if order == "turns":
        turn = [i for n in sections for i in range(n)]
        axis = [a for _, a in sorted(zip(turn, axis))]
    return axis


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    state = {"op": case["op"], "backward": case["backward"]}
    if case["op"] == "rope_axes":
        B, T, d, rows = case["batch"], case["tokens"], case["head_dim"], case["rows"]
        sections = _sections(case)
        # the table that a program builds once: every row's angles, in 64 bits before they are rounded
        angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * \
            torch.pow(10000.0, -torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)[None, :]
        state.update(q=randn(B, T, case["q_heads"], d, dtype=dtype), k=randn(B, T, case["k_heads"], d, dtype=dtype),
                     freqs=torch.stack([angle.cos(), angle.sin()], -1).reshape(rows, d).float(),
                     positions=torch.randint(0, rows, (B, T, len(sections)), generator=gen, device="cuda", dtype=torch.int32),
                     sections=sections, half=case["half"], order=case["order"],
                     pair_axis=torch.tensor(_pair_axis(sections, case["order"]), device="cuda"))
    elif case["op"] == "dropout":
        shape = (case["rows"], case["width"])
        state.update(x=randn(*shape, dtype=dtype), p=case["p"], residual=randn(*shape, dtype=dtype) if case["residual"] else None,
                     seed=torch.randint(-2 ** 62, 2 ** 62, (2,), generator=gen, device="cuda"))
    else:
        N, S, C, G = case["batch"], case["pixels"], case["channels"], case["groups"]
        wtype = dtype if case["weights"] == "same" else torch.float32
        x = (randn(N, S, C) * 1.5 + randn(C)).to(dtype)
        state.update(x=x, weight=(1 + 0.2 * randn(C)).to(wtype), bias=(0.2 * randn(C)).to(wtype), groups=G, eps=1e-5,
                     activation=case["activation"])
        if case["backward"]:
            v = x.float().view(N, S, G, C // G)                    # what the forward pass kept
            mean = v.mean((1, 3))
            var = (v - mean[:, None, :, None]).square().mean((1, 3))
            state.update(dout=randn(N, S, C, dtype=dtype), stats=torch.stack([mean, torch.rsqrt(var + 1e-5)], -1).contiguous())
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------

@functools.lru_cache(None)
def _ops():
    from l2_torch_alloc_amd import ops, wrapper
    if not wrapper.sideaware_enabled():
        wrapper.sideaware_init(install_allocator=False)            # the inputs are there already
    return ops


def _run_own(s):
    ops = _ops()
    if s["op"] == "rope_axes":
        rotate = ops.rope_axes_backward_many if s["backward"] else ops.rope_axes_forward_many
        return rotate([s["q"], s["k"]], s["freqs"], s["positions"], s["sections"], half=s["half"], order=s["order"],
                      outs=[torch.empty_like(s["q"]), torch.empty_like(s["k"])])
    if s["op"] == "dropout":
        if s["backward"]:
            return ops.dropout_backward(s["x"], s["p"], s["seed"])
        return ops.dropout_forward(s["x"], s["p"], s["seed"], residual=s["residual"])
    if s["backward"]:
        return ops.group_norm_backward(s["dout"], s["x"], s["weight"], s["bias"], s["stats"], s["groups"], activation=s["activation"])
    return ops.group_norm_forward(s["x"], s["weight"], s["bias"], s["groups"], eps=s["eps"], activation=s["activation"])


def _rotate(x, cos, sin, half, backward):
    a = x.float()
    first, second = (a.chunk(2, -1) if half else (a[..., 0::2], a[..., 1::2]))
    sin = -sin if backward else sin
    y1, y2 = first * cos - second * sin, first * sin + second * cos
    y = torch.cat([y1, y2], -1) if half else torch.stack([y1, y2], -1).flatten(-2)
    return y.to(x.dtype)


def _philox_round(state):
    """One round of Philox4x32 on counters held in 64-bit integers (products wrap, their halves are right all the same)."""
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    low = 0xFFFFFFFF
    return (b >> 32) & low ^ c1 ^ k0, b & low, (a >> 32) & low ^ c3 ^ k1, a & low, (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low


def _random_halfwords(count, seed):
    """16 random bits for each element: element e has halfword e % 8 of the block of counter (e / 8, offset)."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, device=seed.device)
    key, offset = seed[0], seed[1]
    state = (block & low, block >> 32, (offset & low).expand_as(block), ((offset >> 32) & low).expand_as(block), key & low, (key >> 32) & low)
    words = torch.stack(functools.reduce(lambda st, _: _philox_round(st), range(7), state)[:4], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:count]


def _run_plain(s):
    if s["op"] == "rope_axes":
        pairs = s["q"].shape[-1] // 2
        row = s["positions"].long()[..., s["pair_axis"]]                           # (B, T, pairs)
        cs = s["freqs"].view(-1, pairs, 2)[row, torch.arange(pairs, device=row.device)][:, :, None]
        return [_rotate(x, cs[..., 0], cs[..., 1], s["half"], s["backward"]) for x in (s["q"], s["k"])]
    if s["op"] == "dropout":
        x = s["x"]
        threshold = int(math.floor(s["p"] * 65536 + 0.5))
        keep = (_random_halfwords(x.numel(), s["seed"]) >= threshold).view(x.shape)
        y = torch.where(keep, x.float() * (65536.0 / (65536 - threshold)), torch.zeros((), device=x.device))
        return (y if s["residual"] is None else s["residual"].float() + y).to(x.dtype)
    x, G = s["x"], s["groups"]
    N, S, C = x.shape
    v = x.float().view(N, S, G, C // G)
    w, b = s["weight"].float().view(G, C // G), s["bias"].float().view(G, C // G)
    if not s["backward"]:
        mean = v.mean((1, 3))
        var = (v - mean[:, None, :, None]).square().mean((1, 3))
        rstd = 1.0 / torch.sqrt(var + s["eps"])
        z = (v - mean[:, None, :, None]) * rstd[:, None, :, None] * w + b
        y = z / (1.0 + torch.exp(-z)) if s["activation"] == "silu" else z
        return [y.view(N, S, C).to(x.dtype), torch.stack([mean, rstd], -1)]
    mean, rstd = s["stats"][:, None, :, None, 0], s["stats"][:, None, :, None, 1]
    h = (v - mean) * rstd
    g = s["dout"].float().view(N, S, G, C // G)
    if s["activation"] == "silu":
        z = h * w + b
        sig = 1.0 / (1.0 + torch.exp(-z))
        g = g * (sig * (1.0 + z * (1.0 - sig)))
    gw = g * w
    dx = rstd * (gw - gw.mean((1, 3), keepdim=True) - h * (gw * h).mean((1, 3), keepdim=True))
    return [dx.view(N, S, C).to(x.dtype), (g * h).sum((0, 1)).view(C).to(s["weight"].dtype), g.sum((0, 1)).view(C).to(s["bias"].dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "rope_axes":
        tokens, d = case["batch"] * case["tokens"], case["head_dim"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * d
        table = min(case["rows"], tokens) * d * 4                  # each row that occurs, once
        return {"bytes": 2 * values * size + table + 4 * tokens * len(_sections(case)), "flops": 3 * values}
    if case["op"] == "dropout":
        values = case["rows"] * case["width"]
        return {"bytes": values * size * (3 if case["residual"] else 2), "flops": 2 * values}
    values = case["batch"] * case["pixels"] * case["channels"]
    small = case["channels"] * (16 if case["backward"] else 8) + case["batch"] * case["groups"] * 8
    return {"bytes": values * size * (3 if case["backward"] else 2) + small, "flops": values * (24 if case["backward"] else 14)}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope_axes":
        # every pair as a complex number, turned by its angle
        d = case["head_dim"]
        cs = torch.view_as_complex(s["freqs"].double().view(-1, d // 2, 2).contiguous())
        axis = _pair_axis(s["sections"], s["order"])
        turned = []
        for x in (s["q"], s["k"]):
            v = x.double()
            v = torch.stack([v[..., :d // 2], v[..., d // 2:]], -1) if s["half"] else v.view(*v.shape[:-1], d // 2, 2)
            v = torch.view_as_complex(v.contiguous())
            for j in range(d // 2):
                turn = cs[s["positions"][..., axis[j]].long(), j]
                v[..., j] *= (turn.conj() if s["backward"] else turn)[..., None]
            y = torch.view_as_real(v)
            turned.append(torch.cat([y[..., 0], y[..., 1]], -1) if s["half"] else y.flatten(-2))
        return turned
    if case["op"] == "dropout":
        # the generator in numpy's unsigned integers
        import numpy as np
        count = case["rows"] * case["width"]
        key, offset = (int(v) & (2 ** 64 - 1) for v in s["seed"].tolist())
        block = np.arange((count + 7) // 8, dtype=np.uint64)
        mask = np.uint64(0xFFFFFFFF)
        w = [block & mask, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
        for i in range(7):
            k = [np.uint64((key + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((key >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)]
            m0, m1 = np.uint64(0xD2511F53) * w[0], np.uint64(0xCD9E8D57) * w[2]
            w = [(m1 >> np.uint64(32)) ^ w[1] ^ k[0], m1 & mask, (m0 >> np.uint64(32)) ^ w[3] ^ k[1], m0 & mask]
        bits = np.empty((block.size, 8), dtype=np.uint16)
        for i in range(4):
            bits[:, 2 * i], bits[:, 2 * i + 1] = w[i] & np.uint64(0xFFFF), w[i] >> np.uint64(16)
        dropped = math.floor(case["p"] * 65536 + 0.5)
        kept = torch.from_numpy(bits.reshape(-1)[:count].astype(np.int32) >= dropped).to("cuda").view(s["x"].shape)
        y = kept.double() * s["x"].double() / (1.0 - dropped / 65536.0)
        return y if s["residual"] is None else y + s["residual"].double()
    N, S, C, G = case["batch"], case["pixels"], case["channels"], case["groups"]
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    spread = lambda t: t.repeat_interleave(C // G, -1)[:, None]                    # (N, G) -> (N, 1, C)  # noqa: E731
    pool = lambda t: t.sum(1).view(N, G, C // G).sum(-1) / (S * (C // G))          # (N, S, C) -> (N, G)  # noqa: E731
    if not case["backward"]:
        mean = pool(x)
        rstd = (pool((x - spread(mean)) ** 2) + s["eps"]) ** -0.5
        z = w * (x - spread(mean)) * spread(rstd) + b
        return [z * torch.sigmoid(z) if s["activation"] == "silu" else z, torch.stack([mean, rstd], -1)]
    mean, rstd = spread(s["stats"][..., 0].double()), spread(s["stats"][..., 1].double())
    h, g = (x - mean) * rstd, s["dout"].double()
    if s["activation"] == "silu":
        z = w * h + b
        g = g * (torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z))
    return [rstd * (w * g - spread(pool(w * g)) - h * spread(pool(w * g * h))), (g * h).sum((0, 1)), g.sum((0, 1))]
