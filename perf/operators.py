"""Cases of the packed-batch operators: row maps of a batch of images and clips,
rotary positions with several axes, and attention with capped scores, distance
bias, document, causal and prefix masks.

``run`` computes a case in plain torch operations, or, with ``own`` true, by
the calls a user makes of ``beatlm_b200.ops``."""
import math

import torch

own = False

HD = 64  # the attention kernels' head width


def listed():
    return [
        # eight pictures of different sizes in one request, patches of 14 px: the smallest batch
        {"name": "pack_album", "op": "pack", "images": 8, "side": 37, "frames": 1, "lead": 1,
         "slack": 64, "normalized": False},
        # a server's batch of a thousand pictures and short clips
        {"name": "pack_server", "op": "pack", "images": 1021, "side": 50, "frames": 4, "lead": 0,
         "slack": 4096, "normalized": True},
        # one new token of each of eight streams: Q and K of 16 heads, time/height/width axes
        {"name": "rope_tokens", "op": "rope", "rows": 8, "heads": 32, "head_dim": 64, "axes": 3,
         "dtype": "f16", "pairing": "half", "inverse": False},
        # one 518 px frame of the small encoder: Q and K of 6 heads, two axes
        {"name": "rope_frame", "op": "rope", "rows": 1370, "heads": 12, "head_dim": 64, "axes": 2,
         "dtype": "bf16", "pairing": "axis_half", "inverse": False},
        # a batch of clips through the large encoder
        {"name": "rope_clips", "op": "rope", "rows": 60280, "heads": 32, "head_dim": 64, "axes": 3,
         "dtype": "bf16", "pairing": "half", "inverse": False},
        # the inverse rotation of f32 rows, a head width that is no power of two
        {"name": "rope_inverse", "op": "rope", "rows": 5477, "heads": 16, "head_dim": 80, "axes": 2,
         "dtype": "f32", "pairing": "adjacent", "inverse": True},
        # seven pictures of different sizes through the small encoder: document mask alone
        {"name": "attn_album", "op": "attn", "form": "packed", "seqs": 7, "tokens": 1370, "heads": 6,
         "kv_heads": 6, "qk": "bf16", "last_rows": 0, "mask": "none", "cap": 0.0, "bias": "none"},
        # pictures through the large encoder, scores capped, bias by distance on the patch grid
        {"name": "attn_capped", "op": "attn", "form": "packed", "seqs": 8, "tokens": 1600,
         "heads": 16, "kv_heads": 16, "qk": "bf16", "last_rows": 0, "mask": "none", "cap": 30.0,
         "bias": "grid"},
        # a text-and-image sequence: causal behind a prefix that sees itself whole, bias by distance
        {"name": "attn_prefix", "op": "attn", "form": "padded", "seqs": 2, "tokens": 5477,
         "heads": 12, "kv_heads": 4, "qk": "f16", "last_rows": 0, "mask": "prefix", "cap": 0.0,
         "bias": "index"},
        # a clip of eight 518 px frames seen whole by the large encoder
        {"name": "attn_clip", "op": "attn", "form": "padded", "seqs": 1, "tokens": 10960,
         "heads": 16, "kv_heads": 16, "qk": "bf16", "last_rows": 0, "mask": "none", "cap": 0.0,
         "bias": "none"},
        # the newest token of sixteen streams over what they have kept
        {"name": "attn_token", "op": "attn", "form": "padded", "seqs": 16, "tokens": 8192,
         "heads": 16, "kv_heads": 8, "qk": "bf16", "last_rows": 1, "mask": "causal", "cap": 50.0,
         "bias": "index"},
        # the newest frame of two streams over the frames before it
        {"name": "attn_frame", "op": "attn", "form": "padded", "seqs": 2, "tokens": 5480,
         "heads": 6, "kv_heads": 6, "qk": "f16", "last_rows": 1370, "mask": "causal", "cap": 0.0,
         "bias": "none"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pack", "rope", "rope", "attn", "attn", "attn"])
    if op == "pack":
        return {"op": "pack", "images": _log(rng, 4, 1000), "side": rng.randint(8, 50),
                "frames": rng.randint(1, 4), "lead": rng.randint(0, 5), "slack": _log(rng, 1, 4000),
                "normalized": rng.random() < 0.5}
    if op == "rope":
        heads, head_dim = rng.randint(1, 32), rng.choice([32, 48, 64, 72, 80, 96, 128, 256])
        most = 60280 * 32 * 64 // (heads * head_dim * 2)
        return {"op": "rope", "rows": _log(rng, 1, min(60000, most)), "heads": heads,
                "head_dim": head_dim, "axes": rng.randint(1, 3),
                "dtype": rng.choice(["f16", "bf16", "f32"]),
                "pairing": rng.choice(["half", "adjacent", "axis_half"]),
                "inverse": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 6, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 16])
    form = rng.choice(["packed", "padded"])
    last = 0 if form == "packed" else rng.choice([0, 0, 1, 1, rng.randint(2, 16),
                                                  _log(rng, 17, 1400)])
    if last == 0:
        tokens = _log(rng, 1, 5400)
        seqs = rng.randint(1, max(1, min(24, 10960 ** 2 * 16 // (4 * tokens * tokens * heads))))
    else:
        tokens = _log(rng, max(1, last), 8192)
        seqs = rng.randint(1, 16 if last < 64 else 2)
    return {"op": "attn", "form": form, "seqs": seqs, "tokens": tokens, "heads": heads,
            "kv_heads": kv, "qk": rng.choice(["f16", "bf16"]), "last_rows": last,
            "mask": rng.choice(["none", "causal", "prefix"]),
            "cap": rng.choice([0.0, 0.0, round(rng.uniform(5.0, 50.0), 1)]),
            "bias": rng.choice(["none", "index", "grid"])}


# ------------------------------------------------------------------ inputs

def _sizes(case):
    """The batch's sizes (t, h, w), most of them single frames; their order is prepare()'s."""
    g = torch.Generator().manual_seed(case["images"])
    n, side = case["images"], case["side"]
    hw = torch.randint(1, side + 1, (n, 2), generator=g)
    t = torch.randint(1, case["frames"] + 1, (n, 1), generator=g)
    t = torch.where(torch.rand((n, 1), generator=g) < 0.7, torch.ones_like(t), t)
    return torch.cat([t, hw], 1)


def _rows(case):
    return int((_sizes(case).prod(1) + case["lead"]).sum()) + case["slack"]


def _positions(rows, axes, g):
    """(t, y, x) of rows that walk through frames of 37 x 37 patches from a far frame on."""
    first = torch.randint(0, 100000, (1,), generator=g)
    r = torch.arange(rows) + first * 1369 + torch.randint(0, 1369, (1,), generator=g)
    p = torch.stack([r // 1369, r // 37 % 37, r % 37], 1)
    return p[:, 3 - axes:].to(torch.float32).contiguous()


def _lengths(case):
    """Rows of each sequence: spread over a tenth to all of `tokens`, the first one whole."""
    t = case["tokens"]
    lo = max(1, t // 10)
    return [t - int((t - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(case["seqs"])]


def _sections(case):
    """Pairs of each axis: as even as they go, the later axes taking what is left."""
    pairs, axes = case["head_dim"] // 2, case["axes"]
    return [pairs * (a + 1) // axes - pairs * a // axes for a in range(axes)]


def _pairs(case):
    """(axis, frequency, low element, high element) of each pair; 64-bit frequencies."""
    sections, pairs = _sections(case), case["head_dim"] // 2
    n = torch.tensor(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), n)
    first = (torch.cumsum(n, 0) - n)[axis]
    j = torch.arange(pairs)
    freq = torch.pow(torch.tensor(100.0, dtype=torch.float64), -(j - first).double() / n[axis])
    low = {"half": j, "adjacent": 2 * j, "axis_half": first + j}[case["pairing"]]
    high = low + {"half": pairs, "adjacent": 1, "axis_half": n[axis]}[case["pairing"]]
    return axis.cuda(), freq.cuda(), low.cuda(), high.cuda()


def prepare(case, seed):
    g = torch.Generator().manual_seed(int(seed))
    d = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "pack":
        grids, rows = _sizes(case)[torch.randperm(case["images"], generator=g)], _rows(case)
        turned = torch.rand((case["images"], 1), generator=g) < 0.5  # upright or not
        grids = torch.where(turned, grids[:, [0, 2, 1]], grids)
        s["grids"], s["capacity"] = grids.to(torch.int32).cuda(), rows
        s["offsets"] = torch.zeros(case["images"] + 1, dtype=torch.int32, device="cuda")
        s["image"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["positions"] = torch.zeros((rows, 3), dtype=torch.float32, device="cuda")
        return s
    if case["op"] == "rope":
        dt = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[case["dtype"]]
        x = torch.randn((case["rows"], case["heads"], case["head_dim"]), generator=d, device="cuda")
        s["x"], s["out"] = x.to(dt), torch.empty_like(x, dtype=dt)
        s["positions"] = _positions(case["rows"], case["axes"], g).cuda()
        s["pairs"] = _pairs(case)  # the plain form's tables
        return s
    n, t, h, kv = case["seqs"], case["tokens"], case["heads"], case["kv_heads"]
    length = torch.tensor(_lengths(case))
    if case["form"] == "packed":
        begin = torch.cumsum(length, 0) - length
        rows = int(length.sum()) + 16  # rows behind the last sequence
        s["offsets"] = torch.cat([begin, length.sum()[None]]).to(torch.int32).cuda()
    else:
        begin, rows = torch.arange(n) * t, n * t
        s["lengths"] = length.to(torch.int32).cuda()
    qkv = torch.empty((rows, h + 2 * kv, HD), dtype=torch.int16, device="cuda")
    qk = torch.randn((rows, h + kv, HD), generator=d, device="cuda")
    qk[:, :, 0] += 1.0  # scores around a mean above zero, as trained heads have
    qkv[:, :h + kv] = qk.to(torch.bfloat16 if case["qk"] == "bf16" else torch.float16).view(torch.int16)
    v = torch.randn((rows, kv, HD), generator=d, device="cuda")
    qkv[:, h + kv:] = v.to(torch.float16).view(torch.int16)
    s["qkv"] = qkv
    s["out"] = torch.zeros((rows, h * HD), dtype=torch.bfloat16, device="cuda")
    if case["mask"] == "prefix":
        s["prefix"] = (length // 4).to(torch.int32).cuda()
    if case["bias"] != "none":
        s["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, h + 1, device="cuda") / h).float()
    if case["bias"] == "grid":
        s["positions"] = _positions(rows, 2, g).cuda()
    # the plain form's index tables: key rows and query rows of each sequence, padded
    most = int(length.max())
    r = case["last_rows"] or most
    k = torch.arange(most)[None].expand(n, -1)
    q = length[:, None] - r + torch.arange(r)[None] if case["last_rows"] else k
    kok, qok = k < length[:, None], (q >= 0) & (q < length[:, None])
    clip = lambda i: torch.minimum(i.clamp(min=0), length[:, None] - 1)  # noqa: E731
    s["k_at"], s["q_at"] = clip(k).cuda(), clip(q).cuda()
    s["k_row"], s["q_row"] = (clip(k) + begin[:, None]).cuda(), (clip(q) + begin[:, None]).cuda()
    s["k_ok"] = kok.cuda()
    s["picked"] = torch.nonzero(qok.reshape(-1))[:, 0].cuda()
    s["written"] = (clip(q) + begin[:, None])[qok].cuda()
    return s


# ------------------------------------------------------------------ a pass

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _plain_pack(s):
    case, grids, rows = s["case"], s["grids"].long(), s["capacity"]
    count = grids.prod(1) + case["lead"]
    ends = torch.cumsum(count, 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    r = torch.arange(rows, device=grids.device)
    image = torch.searchsorted(ends, r, right=True)
    real = image < grids.shape[0]
    at = image.clamp(max=grids.shape[0] - 1)
    g = grids[at]
    p = r - offsets[at] - case["lead"]
    c = torch.stack([p // (g[:, 1] * g[:, 2]), p // g[:, 2] % g[:, 1], p % g[:, 2]], 1)
    pos = ((2 * c + 1 - g).float() / g.float()) if case["normalized"] else c.float()
    pos = torch.where((real & (p >= 0))[:, None], pos, torch.zeros_like(pos))
    return {"offsets": offsets.to(torch.int32), "positions": pos,
            "image": torch.where(real, image, torch.full_like(image, -1)).to(torch.int32)}


def _plain_rope(s):
    case, x = s["case"], s["x"].float()
    axis, freq, low, high = s["pairs"]
    angle = s["positions"].double()[:, axis] * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    sin = -sin if case["inverse"] else sin
    a, b = x[:, :, low], x[:, :, high]
    y = torch.empty_like(x)
    y[:, :, low] = a * cos - b * sin
    y[:, :, high] = b * cos + a * sin
    return y.to(s["x"].dtype)


def _heads(s):
    """Q, K, V of every row in 32 bits."""
    case, t = s["case"], s["qkv"]
    h, kv = case["heads"], case["kv_heads"]
    qk = t[:, :h + kv].view(torch.bfloat16 if case["qk"] == "bf16" else torch.float16).float()
    return qk[:, :h], qk[:, h:], t[:, h + kv:].view(torch.float16).float()


def _plain_attn(s):
    case = s["case"]
    h, kv = case["heads"], case["kv_heads"]
    q, k, v = _heads(s)
    q = q[s["q_row"]].transpose(1, 2)  # [seqs, heads, rows, 64]
    k = k[s["k_row"]].transpose(1, 2).repeat_interleave(h // kv, 1)
    v = v[s["k_row"]].transpose(1, 2).repeat_interleave(h // kv, 1)
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(HD))
    if case["cap"]:
        x.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["bias"] == "index":
        far = (s["q_at"][:, :, None] - s["k_at"][:, None]).abs().float()
        x -= s["slopes"][None, :, None, None] * far[:, None]
    if case["bias"] == "grid":
        p, o = s["positions"][s["q_row"]][:, :, None], s["positions"][s["k_row"]][:, None]
        far = ((p[..., 0] - o[..., 0]).square() + (p[..., 1] - o[..., 1]).square()).sqrt()
        x -= s["slopes"][None, :, None, None] * far[:, None]
    seen = s["k_ok"][:, None, :]
    if case["mask"] != "none":
        back = s["k_at"][:, None] <= s["q_at"][:, :, None]
        if case["mask"] == "prefix":
            back = back | (s["k_at"][:, None] < s["prefix"][:, None, None])
        seen = seen & back
    x.masked_fill_(~seen[:, None], float("-inf"))
    x.sub_(x.amax(3, keepdim=True)).exp_()
    o = (x @ v) / x.sum(3, keepdim=True)
    out = s["out"].zero_()
    o = o.transpose(1, 2).reshape(-1, h * HD)
    out[s["written"]] = o[s["picked"]].to(out.dtype)
    return out


def _own_pack(s):
    from beatlm_b200 import ops
    case = s["case"]
    ops.pack(s["grids"], offsets=s["offsets"], image=s["image"], positions=s["positions"],
             lead=case["lead"], normalized=case["normalized"])
    return {"offsets": s["offsets"], "positions": s["positions"], "image": s["image"]}


def _own_rope(s):
    from beatlm_b200 import ops
    case = s["case"]
    return ops.rope(s["x"], s["positions"], sections=_sections(case), theta=100.0,
                    pairing=case["pairing"], inverse=case["inverse"], out=s["out"])


def _own_attn(s):
    from beatlm_b200 import ops
    case = s["case"]
    kw = {"offsets": s["offsets"]} if case["form"] == "packed" else {"lengths": s["lengths"]}
    return ops.masked_attention(
        s["qkv"], heads=case["heads"], kv_heads=case["kv_heads"], qk_dtype=case["qk"],
        last_rows=case["last_rows"], mask=None if case["mask"] == "none" else case["mask"],
        prefix=s.get("prefix"), cap=case["cap"] or None, slopes=s.get("slopes"),
        positions=s.get("positions"), out=s["out"], **kw)


_plain = {"pack": _plain_pack, "rope": _plain_rope, "attn": _plain_attn}
_own = {"pack": _own_pack, "rope": _own_rope, "attn": _own_attn}


# ------------------------------------------------------------------ what a pass needs

def _seen_pairs(case, n):
    """(query, key) pairs of one sequence of n rows."""
    r = min(case["last_rows"] or n, n)
    if case["mask"] == "none":
        return r * n
    first = n - r  # rows first .. n-1 see row + 1 keys each, at least the prefix
    seen = sum(range(first + 1, n + 1))
    if case["mask"] == "prefix":
        p = n // 4
        seen += sum(p - i - 1 for i in range(first, p - 1)) if first < p else 0
    return seen


def work(case):
    if case["op"] == "pack":
        return {"bytes": 16.0 * case["images"] + 16.0 * _rows(case), "flops": 0.0}
    if case["op"] == "rope":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["heads"] * case["head_dim"]
        return {"bytes": 2.0 * n * size + 4.0 * case["rows"] * case["axes"], "flops": 3.0 * n}
    h, kv, lengths = case["heads"], case["kv_heads"], _lengths(case)
    pairs = sum(_seen_pairs(case, m) for m in lengths)
    rows = sum(min(case["last_rows"] or m, m) for m in lengths)
    return {"bytes": 2.0 * HD * (2 * h * rows + 2 * kv * sum(lengths)), "flops": 4.0 * HD * h * pairs}


# ------------------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        offsets, pos, image = [0], [], []
        for i, (t, h, w) in enumerate(s["grids"].tolist()):
            axes = [torch.arange(n, dtype=torch.float64) for n in (t, h, w)]
            if case["normalized"]:
                axes = [(2 * a + 1 - n) / n for a, n in zip(axes, (t, h, w))]
            grid = torch.cartesian_prod(*axes).reshape(-1, 3)
            pos += [torch.zeros((case["lead"], 3), dtype=torch.float64), grid]
            offsets.append(offsets[-1] + case["lead"] + grid.shape[0])
            image += [torch.full((case["lead"] + grid.shape[0],), i)]
        left = s["capacity"] - offsets[-1]
        pos.append(torch.zeros((left, 3), dtype=torch.float64))
        image.append(torch.full((left,), -1))
        return {"offsets": torch.tensor(offsets), "positions": torch.cat(pos),
                "image": torch.cat(image)}
    if case["op"] == "rope":
        x, pos = s["x"].double(), s["positions"].double()
        y, sign, start = torch.empty_like(x), -1.0 if case["inverse"] else 1.0, 0
        for a, n in enumerate(_sections(case)):
            for j in range(n):
                lo, hi = {"half": (start + j, start + j + case["head_dim"] // 2),
                          "adjacent": (2 * (start + j), 2 * (start + j) + 1),
                          "axis_half": (2 * start + j, 2 * start + j + n)}[case["pairing"]]
                z = torch.polar(torch.ones_like(pos[:, a]), sign * pos[:, a] * 100.0 ** (-j / n))
                z = torch.complex(x[:, :, lo], x[:, :, hi]) * z[:, None]
                y[:, :, lo], y[:, :, hi] = z.real, z.imag
            start += n
        return y
    h, kv = case["heads"], case["kv_heads"]
    t = s["qkv"]
    qk = t[:, :h + kv].view(torch.bfloat16 if case["qk"] == "bf16" else torch.float16).double()
    v = t[:, h + kv:].view(torch.float16).double()
    if case["form"] == "packed":
        ends = s["offsets"].tolist()
        spans = list(zip(ends[:-1], ends[1:]))
    else:
        spans = [(i * case["tokens"], i * case["tokens"] + n)
                 for i, n in enumerate(s["lengths"].tolist())]
    out = torch.zeros((t.shape[0], h * HD), dtype=torch.float64, device="cuda")
    for i, (b, e) in enumerate(spans):
        n = e - b
        first = max(0, n - case["last_rows"]) if case["last_rows"] else 0
        rows, keys = torch.arange(first, n, device="cuda"), torch.arange(n, device="cuda")
        hidden = None
        if case["mask"] != "none":
            p = int(s["prefix"][i]) if case["mask"] == "prefix" else 0
            hidden = keys[None] >= torch.clamp(rows + 1, min=p)[:, None]
        if case["bias"] == "index":
            far = (rows[:, None] - keys[None]).abs().double()
        elif case["bias"] == "grid":
            p = s["positions"][b:e].double()
            far = torch.hypot(p[first:, 0][:, None] - p[:, 0], p[first:, 1][:, None] - p[:, 1])
        for j in range(h):
            x = qk[b + first:e, j] @ qk[b:e, h + j // (h // kv)].T / 8.0
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["bias"] != "none":
                x -= s["slopes"][j].double() * far
            if hidden is not None:
                x[hidden] = float("-inf")
            out[b + first:e, j * HD:(j + 1) * HD] = torch.softmax(x, 1) @ v[b:e, j // (h // kv)]
    return out
