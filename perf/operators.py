"""The conditioning operators of a denoiser step, with their plain forms: what is measured and on which sizes.

* `context`  attention of query tokens to an encoder's states of another length (`context_attention`)
* `shared`   the same where the whole batch shares a long run of states (`shared_context_attention`)
* `w4`       linear layers with 4-bit weights and group scales for a few rows (`w4.w4_linear`)

`run` computes them in plain fp32 torch operations, or, with `own` set, through this repository's entry points.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attn(name, op, b, lq, h, hkv, d, lkv, dtype, valid, ls=0):
    case = {"op": op, "b": b, "lq": lq, "h": h, "hkv": hkv, "d": d, "lkv": lkv, "dtype": dtype, "valid": valid}
    if op == "shared":
        case["ls"] = ls
    return {"name": name, **case} if name else case


def _w4(name, m, n, k, group, dtype, act, bias):
    case = {"op": "w4", "m": m, "n": n, "k": k, "group": group, "dtype": dtype, "act": act, "bias": bias}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one query token (a pooled readout) against a 256-token prompt and its duration token: the smallest call
        _attn("context_one_token", "context", 1, 1, 16, 16, 64, 257, "bf16", "all"),
        # the DiT's cross attention for a 120 s clip pair: a padded prompt, its duration token behind the padding
        _attn("context_dit_120s", "context", 2, 2648, 16, 16, 64, 257, "bf16", "holes"),
        # a ragged batch with grouped kv heads, one clip without any context, unset rows behind each length
        _attn("context_ragged", "context", 3, 647, 12, 4, 128, 1421, "fp16", "lens"),
        # a 120 s clip pair conditioned on the latents of a 380 s recording: the largest attention
        _attn("context_recording", "context", 2, 2648, 16, 16, 64, 8184, "bf16", "all"),
        # one token for each of 8 sequences against long contexts, grouped kv heads: the serving form
        _attn("context_long_token", "context", 8, 1, 16, 4, 64, 32768, "bf16", "all"),
        # eight variations of one clip that share a 120 s reference recording, each with a prompt of its own
        _attn("shared_variations", "shared", 8, 646, 16, 16, 64, 128, "bf16", "holes", ls=2584),
        # one token for each of 32 sequences behind a long common prefix
        _attn("shared_long_token", "shared", 32, 1, 16, 4, 64, 257, "bf16", "lens", ls=16384),
        # a handful of tokens, short odd lengths
        _attn("shared_short", "shared", 4, 17, 8, 8, 128, 33, "fp16", "lens", ls=201),
        # the timestep embedder of a clip pair: Fourier features to the model width, SiLU
        _w4("w4_timestep", 2, 1024, 256, 128, "bf16", "silu", False),
        # the adaLN projection of a clip pair: six vectors of the model width
        _w4("w4_adaln", 2, 6144, 1024, 128, "bf16", "none", True),
        # a wide layer for one row: bound by the weights' bytes
        _w4("w4_wide_row", 1, 16384, 8192, 128, "bf16", "none", False),
        # thirteen rows, an odd number of outputs, small groups
        _w4("w4_odd_rows", 13, 8201, 4096, 32, "fp16", "none", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["context", "shared", "w4"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "w4":
        group = rng.choice([32, 64, 128])
        return _w4(None, _log(rng, 1, 32), _log(rng, 256, 16384), group * _log(rng, 256 // group, 8192 // group), group,
                   dtype, rng.choice(["none", "silu"]), rng.random() < 0.5)
    hkv = rng.choice([1, 2, 4, 8, 12, 16])
    h = hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if hkv * g <= 24])
    d = rng.choice([64, 128])
    valid = rng.choice(["all", "lens", "holes"])
    if op == "context":
        b, lq, lkv, ls = rng.randint(1, 8), _log(rng, 1, 2648), _log(rng, 1, 32768), 0
    else:
        b, lq, lkv, ls = _log(rng, 2, 32), _log(rng, 1, 646), _log(rng, 1, 1024), _log(rng, 16, 16384)
    while b * h * lq * (lkv + ls) * d > 4e10:  # below the largest listed call, and the plain form's scores in memory
        if b > 2:
            b //= 2
        elif ls > lkv:
            ls //= 2
        else:
            lkv, lq = max(1, lkv // 2), max(1, (lq * 3) // 4)
    return _attn(None, op, b, lq, h, hkv, d, lkv, dtype, valid, ls=ls)


def _own_valid(case, device="cpu"):
    """Which of its own states each sequence may read, `(B, Lkv)`, by the case alone."""
    b, lkv = case["b"], case["lkv"]
    j = torch.arange(lkv, device=device)[None, :]
    if case["valid"] == "all":
        return (j >= 0).expand(b, lkv)
    row = torch.arange(b, device=device)[:, None]
    if case["valid"] == "lens":  # lengths spread up to the full one; the first of three or more is empty
        n = lkv * (row + 1) // b
        return j < (n * (row > 0) if b > 2 else n)
    n = 1 + (lkv - 1) * (row + 1) // (b + 2)  # a prompt, padding, and the last state, always there
    return (j < n) | (j == lkv - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "w4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        w = normal(n, k).mul_(1 / math.sqrt(k)).view(n, k // group, group)
        scale = (w.abs().amax(-1, keepdim=True) / 7).bfloat16().float()
        q = torch.round(w / scale).clamp_(-7, 7).to(torch.int16).view(n, k)
        packed, scales = _pack(q, scale.view(n, k // group).bfloat16(), group)
        return {"case": case, "x": normal(m, k).to(dt), "packed": packed, "scales": scales,
                "bias": (0.1 * normal(n)).to(dt) if case["bias"] else None}
    b, lkv, width = case["b"], case["lkv"], case["hkv"] * case["d"]
    valid = _own_valid(case, "cuda")
    kv = normal(b, lkv, 2 * width).to(dt)
    state = {"case": case, "q": normal(b, case["lq"], case["h"] * case["d"]).to(dt), "lens": None, "mask": None}
    if case["valid"] == "lens":  # what lies behind a sequence's length was never written
        state["lens"] = valid.sum(-1).int()
        kv.masked_fill_(~valid[..., None], float("nan"))
    elif case["valid"] == "holes":
        state["mask"] = valid.contiguous()
    state["kv"] = kv
    if case["op"] == "shared":
        state["shared_kv"] = normal(case["ls"], 2 * width).to(dt)
    return state


# ---- 4-bit weights: per 16 outputs x 128 inputs one 1,024-byte block. Byte 512 * (r // 8) + 64 * (r % 8) + 16 * t
# + 4 * w begins the 32-bit word of output r and inputs 32 w + 8 t .. + 8; its nibbles, lowest first, are the inputs
# 0, 2, 4, 6, 1, 3, 5, 7 of those eight, each value + 8. Scales: per block (128 / group, 16) in bf16.
_NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]


def _pack(q, scale, group):
    n, k = q.shape
    nt, kb = -(-n // 16), -(-k // 128)
    full = torch.zeros(nt * 16, kb * 128, dtype=torch.int16, device=q.device)
    full[:n, :k] = q
    #                 tile, half, row, block, w, t, eight -> tile, block, half, row, t, w, eight
    x = (full + 8).view(nt, 2, 8, kb, 4, 4, 8).permute(0, 3, 1, 2, 5, 4, 6)[..., _NIBBLES]
    x = x.to(torch.uint8)
    packed = (x[..., 0::2] | (x[..., 1::2] << 4)).reshape(nt, kb, 1024).contiguous()
    sc = torch.zeros(nt * 16, kb * 128 // group, dtype=torch.bfloat16, device=q.device)
    sc[:n, :k // group] = scale
    return packed, sc.view(nt, 16, kb, 128 // group).permute(0, 2, 3, 1).contiguous()


def _unpack(packed, scales, n, k):
    """The integers `(n, k)` in fp32 and the scales `(n, groups)`."""
    nt, kb, _ = packed.shape
    by = packed.view(nt, kb, 2, 8, 4, 4, 4)
    x = torch.stack([by & 15, by >> 4], -1).flatten(-2)  # nibbles, lowest first
    back = torch.empty_like(x)
    back[..., _NIBBLES] = x
    q = back.permute(0, 2, 3, 1, 5, 4, 6).reshape(nt * 16, kb * 128)[:n, :k].float() - 8
    s = scales.permute(0, 3, 1, 2).reshape(nt * 16, -1)[:n]
    return q, s


def _heads(x, count, d):
    return x.unflatten(-1, (count, d)).transpose(-3, -2)  # (..., count, length, d)


def _plain_attention(s):
    case = s["case"]
    b, lq, h, hkv, d = case["b"], case["lq"], case["h"], case["hkv"], case["d"]
    q = _heads(s["q"].float(), h, d).reshape(b, hkv, h // hkv * lq, d)  # a kv head's query heads as one run of rows
    k, v = (_heads(t, hkv, d) for t in s["kv"].float().chunk(2, -1))
    valid = torch.ones(b, case["lkv"], dtype=torch.bool, device=q.device)
    if s["lens"] is not None:
        valid = torch.arange(case["lkv"], device=q.device)[None, :] < s["lens"][:, None]
    if s["mask"] is not None:
        valid = valid & s["mask"]
    v = torch.where(valid[:, None, :, None], v, 0.0)  # unset states are not read
    scores = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(~valid[:, None, None, :], -math.inf)
    if case["op"] == "shared":
        ks, vs = (_heads(t, hkv, d) for t in s["shared_kv"].float().chunk(2, -1))
        scores = torch.cat([(q @ ks.transpose(-1, -2)).mul_(d ** -0.5), scores], -1)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    if case["op"] == "shared":
        o = p[..., :case["ls"]] @ vs + p[..., case["ls"]:] @ v
    else:
        o = p @ v
    o = torch.where(total > 0, o / total, 0.0)
    return o.reshape(b, h, lq, d).transpose(1, 2).reshape(b, lq, h * d).to(s["q"].dtype)


def _plain_w4(s):
    case = s["case"]
    q, scale = _unpack(s["packed"], s["scales"], case["n"], case["k"])
    w = (q.unflatten(-1, (-1, case["group"])) * scale[:, :case["k"] // case["group"], None].float()).flatten(-2)
    y = s["x"].float() @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["x"].dtype)


def run(state):
    case = state["case"]
    if own:
        from hummingbird_b200 import context_attention, w4
        if case["op"] == "w4":
            return w4.w4_linear(state["x"], state["packed"], state["scales"], case["n"], case["group"], state["bias"],
                                act=case["act"])
        args = dict(kv_heads=case["hkv"], lens=state["lens"], mask=state["mask"])
        if case["op"] == "shared":
            return context_attention.shared_context_attention(state["q"], state["shared_kv"], state["kv"], case["h"],
                                                              case["d"], **args)
        return context_attention.context_attention(state["q"], state["kv"], case["h"], case["d"], **args)
    return _plain_w4(state) if case["op"] == "w4" else _plain_attention(state)


def work(case):
    if case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k / 2 + 2 * n * k / case["group"] + 2 * m * (n + k) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    own_keys = int(_own_valid(case).sum())
    shared = case.get("ls", 0)
    pairs = case["lq"] * (own_keys + case["b"] * shared)  # per query head
    bytes_ = 2 * 2 * case["b"] * case["lq"] * case["h"] * case["d"] + 4 * (own_keys + shared) * case["hkv"] * case["d"]
    if case["valid"] == "holes":
        bytes_ += case["b"] * case["lkv"]
    elif case["valid"] == "lens":
        bytes_ += 4 * case["b"]
    return {"bytes": bytes_, "flops": 4 * pairs * case["h"] * case["d"]}


def exact(case, seed):
    """By definition in 64 bits: one query head (or one slice of outputs) at a time, only the states that are valid."""
    s = prepare(case, seed)
    if case["op"] == "w4":
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        q, scale = _unpack(s["packed"], s["scales"], case["n"], case["k"])
        group_of = torch.arange(case["k"], device="cuda") // case["group"]
        for a in range(0, case["n"], 2048):
            w = q[a:a + 2048].double() * scale[a:a + 2048].double()[:, group_of]
            y[:, a:a + 2048] = torch.einsum("mk,nk->mn", s["x"].double(), w)
        if s["bias"] is not None:
            y += s["bias"].double()
        return y * torch.special.expit(y) if case["act"] == "silu" else y
    b, lq, h, hkv, d = case["b"], case["lq"], case["h"], case["hkv"], case["d"]
    out = torch.zeros(b, lq, h, d, dtype=torch.float64, device="cuda")
    valid = _own_valid(case, "cuda")
    for i in range(b):
        states = s["kv"][i][valid[i]]
        if case["op"] == "shared":
            states = torch.cat([s["shared_kv"], states])
        states = states.view(-1, 2, hkv, d)
        if not states.shape[0]:
            continue
        for j in range(h):
            key, value = states[:, 0, j * hkv // h].double(), states[:, 1, j * hkv // h].double()
            query = s["q"][i].view(lq, h, d)[:, j].double()
            weights = torch.softmax(query @ key.T / math.sqrt(d), -1)
            out[i, :, j] = weights @ value
    return out.view(b, lq, h * d)
