"""Workloads of the attention path around a 4-bit K/V cache, with the plain form of every operator.

The path of one attention layer of a decoder that keeps its cache in 4 bits:

  rope    per-head RMSNorm of queries and keys and the rotary position embedding, one pass
          (attention.qk_norm_rope)
  cache   keys and values quantised into the cache's slots as they are written (Kv4Cache.append),
          then the sequences' positions read back as packed rows (Kv4Cache.read)
  attn4   attention of single new tokens over the cache in 4 bits (Kv4Cache.attend)
  prompt  causal attention of packed prompts or prompt chunks, grouped heads (attention.prompt_attention)

The cache.  A position of one K/V head is head_dim codes of 4 bits (two per byte, the even dimension in
the low half) and head_dim/32 half-precision scales; dimension d belongs to group d mod (head_dim/32) and
stands for (code - 8) * scale.  Writing takes the smallest half with 7 * scale >= max |x| of the group and
rounds x / scale to the nearest code, ties to even.

Lengths: `count` sequences whose lengths fall geometrically from `longest` to `shortest`.
"""
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xiaomi-hexagon-exl3_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from exl3_b200 import attention

    return attention


def lengths(count, longest, shortest):
    if count == 1:
        return [longest]
    return [max(shortest, round(longest * (max(shortest, 1) / longest) ** (i / (count - 1)))) if i < count - 1 else shortest
            for i in range(count)]


def listed():
    return [
        # one decoded token's queries and keys, the decoder's own geometry, far into a long context
        {"name": "rope_token", "op": "rope", "rows": 1, "heads": 16, "kv": 4, "dim": 128, "rotary": 128,
         "interleaved": False, "factor": 1.0, "far": 32768, "dtype": "f32"},
        # a packed prefill step of an odd size: part of the head rotated, interleaved pairs, positions
        # scaled for a context of a million
        {"name": "rope_prompts", "op": "rope", "rows": 8191, "heads": 16, "kv": 4, "dim": 128, "rotary": 64,
         "interleaved": True, "factor": 1.2, "far": 1048576, "dtype": "bf16"},
        # one decoding step of eight requests: a row each into the cache, their contexts read back
        {"name": "cache_step", "op": "cache", "count": 8, "longest": 1, "shortest": 1, "past": 1023, "kv": 4,
         "dim": 128, "dtype": "f32", "read": "f16"},
        # a chunk of a prompt behind a cached start
        {"name": "cache_chunk", "op": "cache", "count": 1, "longest": 512, "shortest": 512, "past": 15361, "kv": 4,
         "dim": 128, "dtype": "f16", "read": "f16"},
        # sixteen whole prompts of ragged lengths, smaller heads
        {"name": "cache_prompts", "op": "cache", "count": 16, "longest": 8192, "shortest": 17, "past": 0, "kv": 8,
         "dim": 64, "dtype": "bf16", "read": "bf16"},
        # one request decoding behind a 512-token prompt, the decoder's own type
        {"name": "attn4_token", "op": "attn4", "rows": 1, "longest": 767, "shortest": 767, "heads": 16, "kv": 4,
         "dim": 128, "dtype": "f32"},
        # one request with a context of 128 k
        {"name": "attn4_long", "op": "attn4", "rows": 1, "longest": 131071, "shortest": 131071, "heads": 16, "kv": 4,
         "dim": 128, "dtype": "bf16"},
        # eight requests between one token and 32 k
        {"name": "attn4_ragged", "op": "attn4", "rows": 8, "longest": 32768, "shortest": 1, "heads": 16, "kv": 4,
         "dim": 128, "dtype": "f16"},
        # a full server: 64 requests, smaller heads, eight queries to a key
        {"name": "attn4_server", "op": "attn4", "rows": 64, "longest": 16384, "shortest": 1000, "heads": 32, "kv": 4,
         "dim": 64, "dtype": "bf16"},
        # a short prompt by itself: latency
        {"name": "prompt_short", "op": "prompt", "count": 1, "longest": 37, "shortest": 37, "past": 0, "heads": 16,
         "kv": 4, "dim": 128, "dtype": "f16", "packed": True},
        # a step of mixed rows: prompt chunks down to single tokens, each behind a cached start
        {"name": "prompt_chunks", "op": "prompt", "count": 7, "longest": 1024, "shortest": 1, "past": 4001, "heads": 16,
         "kv": 4, "dim": 128, "dtype": "f16", "packed": False},
        # one long prompt
        {"name": "prompt_long", "op": "prompt", "count": 1, "longest": 16384, "shortest": 16384, "past": 0, "heads": 16,
         "kv": 4, "dim": 128, "dtype": "bf16", "packed": True},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["rope", "cache", "attn4", "prompt"])
    dim = rng.choice([64, 128, 128])
    heads, kv = rng.choice([(16, 4), (16, 4), (32, 4), (8, 8), (16, 8), (12, 4), (10, 2)])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "rope":
        return {"op": op, "rows": _log(rng, 1, 8191), "heads": heads, "kv": kv, "dim": dim,
                "rotary": rng.choice([dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
                "factor": rng.choice([1.0, 1.0 + round(0.3 * rng.random(), 3)]), "far": _log(rng, 1000, 1048576),
                "dtype": dtype}
    if op == "cache":
        count = _log(rng, 1, 16)
        longest = _log(rng, 1, 8192)
        return {"op": op, "count": count, "longest": longest, "shortest": rng.randint(0, longest) if count > 1 else longest,
                "past": rng.choice([0, _log(rng, 1, 8000)]), "kv": kv, "dim": dim, "dtype": dtype,
                "read": rng.choice(["f32", "f16", "bf16"])}
    if op == "attn4":
        rows = _log(rng, 1, 64)
        longest = _log(rng, 1, 131072 if rows <= 8 else 16384)
        return {"op": op, "rows": rows, "longest": longest, "shortest": rng.randint(1, longest) if rows > 1 else longest,
                "heads": heads, "kv": kv, "dim": dim, "dtype": dtype}
    count = _log(rng, 1, 12)
    longest = _log(rng, 1, 8192 if count == 1 else 2048)
    return {"op": op, "count": count, "longest": longest, "shortest": rng.randint(0, longest) if count > 1 else longest,
            "past": rng.choice([0, 0, _log(rng, 1, 4096)]), "heads": heads, "kv": kv, "dim": dim,
            "dtype": rng.choice(["f16", "bf16"]), "packed": rng.random() < 0.5}


# -- inputs -----------------------------------------------------------------------------------------

def _quantise(x):
    """f32 rows [..., D] -> (codes [..., D/2] uint8, scales [..., D/32] f16)."""
    groups = x.shape[-1] // 32
    x = x.unflatten(-1, (-1, groups))                       # dimension d: [d // groups, d % groups]
    most = x.abs().amax(-2).double()
    scale = torch.minimum(most / 7, torch.tensor(65504.0, dtype=torch.float64, device=x.device)).half()
    low = (scale.double() * 7 < most) & (scale < 65504)
    scale = torch.where(low, (scale.view(torch.int16) + 1).view(torch.float16), scale)
    step = torch.where(scale == 0, torch.ones_like(scale), scale).double().unsqueeze(-2)
    code = (torch.round(x.double() / step).clamp(-7, 7) * (scale != 0).unsqueeze(-2) + 8).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales, type_=torch.float32):
    """What cached positions stand for: codes [..., D/2], scales [..., G] -> [..., D]."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(type_) - 8
    return (code.unflatten(-1, (-1, scales.shape[-1])) * scales.to(type_).unsqueeze(-2)).flatten(-2)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    got = [0]
    for n in lens:
        got.append(got[-1] + n)
    return got


def _filled(lens, kv, dim, max_len, generator):
    """Codes and scales of a cache whose slot s holds lens[s] positions: keys with a few strong channels,
    as rotary keys have, and values around zero."""
    shape = (len(lens), kv, max_len)
    parts = []
    for strong in (6.0, 1.5):
        codes = torch.full(shape + (dim // 2,), 0x88, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(shape + (dim // 32,), dtype=torch.float16, device="cuda")
        channel = 1 + (strong - 1) * (torch.rand(dim, generator=generator, device="cuda") < 0.05)
        for s, n in enumerate(lens):
            if n:
                x = torch.randn((kv, n, dim), generator=generator, device="cuda") * channel
                codes[s, :, :n], scales[s, :, :n] = _quantise(x)
        parts += [codes, scales]
    return parts


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    dim, kv = case["dim"], case["kv"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "rope":
        rows, heads, rotary = case["rows"], case["heads"], case["rotary"]
        # the projections' packed rows [q | k | v]
        qkv = (normal(rows, heads + 2 * kv, dim) * 1.5).to(t)
        state["q"], state["k"] = qkv[:, :heads], qkv[:, heads:heads + kv]
        state["q_weight"], state["k_weight"] = 1 + 0.1 * normal(dim), 1 + 0.1 * normal(dim)
        first = int(torch.randint(0, max(1, case["far"] - rows), (1,), generator=g, device="cuda"))
        state["positions"] = torch.arange(first, first + rows, dtype=torch.int32, device="cuda")
        i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
        state["inv_freq"] = (1e7 ** (-2 * i / rotary)).float()
    elif case["op"] in ("cache", "attn4"):
        count = case["count"] if case["op"] == "cache" else case["rows"]
        lens = lengths(count, case["longest"], case["shortest"])
        past = case.get("past", 0)
        max_len = -(-(max(lens) + past) // 64) * 64
        slots = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
        held = [past] * count if case["op"] == "cache" else [lens[i] for i in slots.argsort().tolist()]
        state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"] = _filled(held, kv, dim, max_len, g)
        state["seq_slot"] = slots
        if case["op"] == "cache":
            rows = sum(lens)
            kvs = (normal(rows, 2 * kv, dim) * 1.5).to(t)
            state["k"], state["v"] = kvs[:, :kv], kvs[:, kv:]
            state["row_seq"] = _ints([s for s, n in enumerate(lens) for _ in range(n)])
            state["row_pos"] = _ints([past + j for n in lens for j in range(n)])
            ends = _offsets([n + past for n in lens])
            state["kv_offsets"], state["total"] = _ints(ends), ends[-1]
        else:
            state["q"] = normal(count, case["heads"], dim).to(t)
            state["row_seq"], state["row_pos"] = _ints(list(range(count))), _ints([n - 1 for n in lens])
        if own:
            state["cache"] = _framework().Kv4Cache.from_tensors(state["k_codes"], state["k_scales"], state["v_codes"],
                                                                state["v_scales"])
    else:
        heads = case["heads"]
        lens = lengths(case["count"], case["longest"], case["shortest"])
        ends = _offsets(lens)
        kv_ends = _offsets([n + case["past"] for n in lens])
        if case["packed"] and not case["past"]:
            qkv = normal(ends[-1], heads + 2 * kv, dim).to(t)
            state["q"], state["k"], state["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        else:
            state["q"] = normal(ends[-1], heads, dim).to(t)
            state["k"], state["v"] = normal(kv_ends[-1], kv, dim).to(t), normal(kv_ends[-1], kv, dim).to(t)
        state["q_offsets"], state["kv_offsets"] = _ints(ends), _ints(kv_ends)
        state["most_q"], state["most_kv"] = max(lens), max(lens) + case["past"]
    return state


# -- the plain forms --------------------------------------------------------------------------------

def _plain_norm_rope(x, weight, angle, s):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    r = s["rotary"]
    rot, rest = y[..., :r], y[..., r:]
    cos = (angle.cos() * s["factor"]).float()[:, None]
    sin = (angle.sin() * s["factor"]).float()[:, None]
    if s["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = rot[..., :r // 2], rot[..., r // 2:]
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rot, rest), -1).to(x.dtype)


def _plain_rope(s):
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    return _plain_norm_rope(s["q"], s["q_weight"], angle, s), _plain_norm_rope(s["k"], s["k_weight"], angle, s)


def _plain_cache(s):
    slot, pos = s["seq_slot"].long()[s["row_seq"].long()], s["row_pos"].long()
    s["k_codes"][slot, :, pos], s["k_scales"][slot, :, pos] = _quantise(s["k"].float())
    s["v_codes"][slot, :, pos], s["v_scales"][slot, :, pos] = _quantise(s["v"].float())
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["kv_offsets"][1:], row, right=True)
    slot, pos = s["seq_slot"].long()[seq], row - s["kv_offsets"].long()[seq]
    t = TYPES[s["read"]]
    return tuple(_values(s[a + "_codes"][slot, :, pos], s[a + "_scales"][slot, :, pos]).to(t) for a in "kv")


def _plain_attn4(s):
    rows, heads, dim = s["q"].shape
    kv, max_len = s["kv"], s["k_codes"].shape[2]
    slot = s["seq_slot"].long()[s["row_seq"].long()]
    k = _values(s["k_codes"][slot], s["k_scales"][slot])                       # [rows, kv, max_len, dim]
    q = s["q"].float().view(rows, kv, heads // kv, dim)
    score = (q @ k.transpose(-1, -2)).mul_(dim ** -0.5)
    score.masked_fill_(torch.arange(max_len, device="cuda") > s["row_pos"].view(-1, 1, 1, 1), float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ _values(s["v_codes"][slot], s["v_scales"][slot])) / total
    return out.reshape(rows, heads, dim).to(s["q"].dtype)


def _plain_prompt(s):
    heads, dim = s["q"].shape[1:]
    kv = s["kv"]
    q0, k0 = s["q_offsets"].long(), s["kv_offsets"].long()
    qn, kn = q0.diff()[:, None], k0.diff()[:, None]
    qi, ki = torch.arange(s["most_q"], device="cuda"), torch.arange(s["most_kv"], device="cuda")
    q_row, k_row = q0[:-1, None] + qi, k0[:-1, None] + ki                      # padded batch of the packed rows
    q = s["q"][q_row.clamp(max=len(s["q"]) - 1)].float()                       # [seq, most_q, heads, dim]
    k, v = (s[a][k_row.clamp(max=len(s[a]) - 1)].float().transpose(1, 2) for a in "kv")  # [seq, kv, most_kv, dim]
    q = q.unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [seq, kv, group * most_q, dim]
    score = (q @ k.transpose(-1, -2)).mul_(dim ** -0.5).unflatten(2, (-1, s["most_q"]))
    seen = (ki <= (qi[:, None] + (kn - qn)[..., None])) & (ki < kn[..., None]) & (qi[:, None] < qn[..., None])
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, s["most_q"])) / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[qi < qn].to(s["q"].dtype)


def run(state):
    s = state
    if own:
        a = _framework()
        if s["op"] == "rope":
            return a.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], eps=EPS,
                                  interleaved=s["interleaved"], attention_factor=s["factor"])
        if s["op"] == "cache":
            s["cache"].append(s["k"], s["v"], s["row_seq"], s["row_pos"], s["seq_slot"])
            return s["cache"].read(s["seq_slot"], s["kv_offsets"], s["total"], dtype=TYPES[s["read"]])
        if s["op"] == "attn4":
            return s["cache"].attend(s["q"], s["row_seq"], s["row_pos"], s["seq_slot"])
        return a.prompt_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["kv_offsets"])
    return {"rope": _plain_rope, "cache": _plain_cache, "attn4": _plain_attn4, "prompt": _plain_prompt}[s["op"]](s)


# -- the least work, and 64 bits ---------------------------------------------------------------------

def work(case):
    dim, kv, b = case["dim"], case["kv"], SIZE[case["dtype"]]
    position = kv * 2 * (dim // 2 + dim // 32 * 2)  # bytes of a cached position, keys and values
    if case["op"] == "rope":
        values = case["rows"] * (case["heads"] + kv) * dim
        return {"bytes": 2 * b * values + 4 * case["rows"] + 8 * dim + 2 * case["rotary"], "flops": 8 * values}
    if case["op"] == "cache":
        lens = lengths(case["count"], case["longest"], case["shortest"])
        rows, past = sum(lens), case["past"] * len(lens)
        return {"bytes": rows * (2 * kv * dim * b + position + 8) + past * position
                + (rows + past) * 2 * kv * dim * SIZE[case["read"]], "flops": 4 * (2 * rows + past) * kv * dim}
    if case["op"] == "attn4":
        lens = lengths(case["rows"], case["longest"], case["shortest"])
        return {"bytes": sum(lens) * position + 2 * case["rows"] * case["heads"] * dim * b,
                "flops": 4 * sum(lens) * case["heads"] * dim}
    lens = lengths(case["count"], case["longest"], case["shortest"])
    rows, past = sum(lens), case["past"]
    pairs = sum(n * past + n * (n + 1) // 2 for n in lens)
    return {"bytes": b * dim * (2 * rows * case["heads"] + 2 * (rows + past * len(lens)) * kv),
            "flops": 4 * pairs * case["heads"] * dim}


def _exact_head(q, k, v, first):
    """Softmax attention in 64 bits: query i of q [n, D] sees keys 0 .. first + i of k, v [m, D]."""
    score = q.double() @ k.double().t()
    score *= q.shape[-1] ** -0.5
    far = torch.arange(len(k), device=q.device) > first + torch.arange(len(q), device=q.device)[:, None]
    score[far] = -torch.inf
    weight = torch.softmax(score, -1)
    return weight @ v.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        outs = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            norm = (x.pow(2).sum(-1) / case["dim"] + EPS).sqrt()
            x = x * w.double() / norm[..., None]
            half = case["rotary"] // 2
            theta = torch.outer(s["positions"].double(), s["inv_freq"].double())
            turn = torch.polar(torch.full_like(theta, case["factor"]), theta)[:, None]
            one = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
            two = one + (1 if case["interleaved"] else half)
            z = torch.complex(x[..., one], x[..., two]) * turn
            x[..., one], x[..., two] = z.real, z.imag
            outs.append(x)
        return tuple(outs)
    if case["op"] == "cache":
        lens = lengths(case["count"], case["longest"], case["shortest"])
        outs = []
        for a in "kv":
            parts, at = [], 0
            for seq, n in enumerate(lens):
                codes = s[a + "_codes"][s["seq_slot"][seq], :, :case["past"]].transpose(0, 1)
                scale = s[a + "_scales"][s["seq_slot"][seq], :, :case["past"]].transpose(0, 1).double()
                groups = scale.shape[-1]
                old = torch.empty(codes.shape[:-1] + (case["dim"],), dtype=torch.float64, device="cuda")
                old[..., 0::2], old[..., 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
                for d in range(groups):
                    old[..., d::groups] *= scale[..., d:d + 1]
                new = s[a][at:at + n].double().clone()
                for d in range(groups):
                    part = new[..., d::groups]
                    top = part.abs().amax(-1, keepdim=True)
                    half = (top / 7).half()
                    # the smallest half that is not below top / 7
                    half = torch.where(half.double() * 7 < top, (half.view(torch.int16) + 1).view(torch.float16), half).double()
                    new[..., d::groups] = torch.where(half > 0, torch.round(part / half.clamp(min=1e-30)) * half, part * 0)
                parts += [old, new]
                at += n
            outs.append(torch.cat(parts))
        return tuple(outs)
    if case["op"] == "attn4":
        rows, heads, dim = s["q"].shape
        share = heads // case["kv"]
        out = torch.empty((rows, heads, dim), dtype=torch.float64, device="cuda")
        for r, n in enumerate(lengths(rows, case["longest"], case["shortest"])):
            for h in range(case["kv"]):
                at = (int(s["seq_slot"][r]), h, slice(0, n))
                k, v = (_values(s[a + "_codes"][at], s[a + "_scales"][at], torch.float64) for a in "kv")
                out[r, h * share:(h + 1) * share] = _exact_head(s["q"][r, h * share:(h + 1) * share], k, v, n)
        return out
    lens = lengths(case["count"], case["longest"], case["shortest"])
    heads = case["heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    q_at = k_at = 0
    for n in lens:
        m = n + case["past"]
        for h in range(heads):
            at = h // (heads // case["kv"])
            out[q_at:q_at + n, h] = _exact_head(s["q"][q_at:q_at + n, h], s["k"][k_at:k_at + m, at], s["v"][k_at:k_at + m, at],
                                                case["past"])
        q_at, k_at = q_at + n, k_at + m
    return out
