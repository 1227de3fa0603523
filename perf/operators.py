"""Performance cases of the training-side operators of a video DiT's attention: the gradients of the dense and of the
gather-KV attention call, and rotary positions with their gradient.

One training step of an attention layer rotates q and k, attends (densely, or each group of query rows to its selected
keys), gets the gradient of the attention output from above and needs dq, dk, dv, which go back through the rotation.
Every case is one call of that chain.  Sizes: the 21 x 39 x 40 latent grid with 24 heads and 2,048 selected tokens, the
head dimensions 64 / 96 / 128 / 144 and the 4,096-token two-head case that the benchmark and the tests use, the 512 text
tokens of a cross-attention, plus short and ragged sequences.

Inputs are clustered latents: a token carries the centroid of its run of neighbouring tokens plus noise; V and the
gradient from above are Gaussian.  Everything comes from the seed alone.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SINKS = 4                      # forced tokens at the start of every index list


def listed():
    return [
        # the smallest dense call: two heads of an odd, short sequence; launch and host latency
        {"name": "dense_small", "kind": "dense", "B": 1, "H": 2, "Lq": 257, "Lk": 257, "D": 64, "dtype": "fp16"},
        # cross-attention of a short clip to its text: few keys, so that the work has to be split over the queries
        {"name": "dense_text", "kind": "dense", "B": 1, "H": 24, "Lq": 4680, "Lk": 512, "D": 128, "dtype": "bf16"},
        # the other head dimension of the sparse dispatch, two clips, ragged lengths
        {"name": "dense_d144", "kind": "dense", "B": 2, "H": 8, "Lq": 4095, "Lk": 4095, "D": 144, "dtype": "fp16"},
        # a dense layer of the single-GPU video DiT
        {"name": "dense_dit", "kind": "dense", "B": 1, "H": 24, "Lq": 32760, "Lk": 32760, "D": 128, "dtype": "bf16"},
        # the smallest sparse call: groups of 64 queries, 512 tokens each
        {"name": "gather_small", "kind": "gather", "B": 1, "H": 2, "L": 4096, "D": 64, "K": 512, "rows": 64, "dtype": "bf16",
         "perm": False, "lengths": False},
        # budgets by mass: every group has a length of its own; ragged, two clips
        {"name": "gather_lengths", "kind": "gather", "B": 2, "H": 6, "L": 4700, "D": 96, "K": 1152, "rows": 128, "dtype": "fp16",
         "perm": True, "lengths": True},
        # a sparse layer of the single-GPU video DiT: most layers of a sparse fine-tuning step are this call
        {"name": "gather_dit", "kind": "gather", "B": 1, "H": 24, "L": 32760, "D": 128, "K": 2048, "rows": 128, "dtype": "bf16",
         "perm": True, "lengths": False},
        # one new token of each of eight sequences at far positions, half layout on half of the head
        {"name": "rope_token", "kind": "rope", "B": 8, "L": 1, "Hq": 24, "Hk": 24, "D": 128, "rot": 64, "axes": 1, "layout": "half",
         "scaling": "yarn", "factor": 8.0, "dtype": "bf16", "backward": False},
        # q and k of the single-GPU video DiT on its three grid axes
        {"name": "rope_dit", "kind": "rope", "B": 1, "L": 32760, "Hq": 24, "Hk": 24, "D": 128, "rot": 128, "axes": 3,
         "layout": "interleaved", "scaling": "none", "factor": 1.0, "dtype": "bf16", "backward": False},
        # the gradient of the same, a longer grid than the model was trained on
        {"name": "rope_dit_bwd", "kind": "rope", "B": 1, "L": 32760, "Hq": 24, "Hk": 24, "D": 128, "rot": 128, "axes": 3,
         "layout": "interleaved", "scaling": "ntk", "factor": 2.0, "dtype": "bf16", "backward": True},
        # gradients in 32 bits, part of the head, half layout, ragged length, fewer key heads
        {"name": "rope_half_bwd", "kind": "rope", "B": 2, "L": 4095, "Hq": 16, "Hk": 4, "D": 144, "rot": 96, "axes": 1,
         "layout": "half", "scaling": "linear", "factor": 4.0, "dtype": "fp32", "backward": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["dense", "dense", "gather", "gather", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "dense":
        Lq = _log(rng, 1, 16380)
        Lk = rng.choice([Lq, _log(rng, 1, 16380), rng.choice([77, 226, 512])])
        B = rng.choice([1, 1, 2])
        return {"kind": kind, "B": B, "H": _log(rng, 1, 24 // B), "Lq": Lq, "Lk": Lk, "D": rng.choice([64, 96, 128, 128, 128, 144]),
                "dtype": dtype}
    if kind == "gather":
        L = _log(rng, 600, 32760)
        B = rng.choice([1, 1, 2])
        rows = 128 if L > 16384 else rng.choice([64, 128, 128])
        K = max(128, min(_log(rng, 128, 2048), L) // 128 * 128)
        return {"kind": kind, "B": B, "H": _log(rng, 1, 24 // B), "L": L, "D": rng.choice([64, 96, 128, 128, 128, 144]), "K": K,
                "rows": rows, "dtype": dtype, "perm": rng.random() < 0.7, "lengths": rng.random() < 0.3}
    D = rng.choice([64, 96, 128, 128, 144])
    axes = rng.choice([1, 1, 3])
    L = _log(rng, 1, 32760)
    Hq = _log(rng, 1, 24)
    return {"kind": kind, "B": rng.choice([1, 1, 2]) if L > 16 else _log(rng, 1, 64), "L": L, "Hq": Hq,
            "Hk": rng.choice([Hq, Hq, max(1, Hq // 4)]), "D": D, "rot": D if axes == 3 else rng.choice([D, D, D // 2, 20]), "axes": axes,
            "layout": rng.choice(["interleaved", "half"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
            "factor": rng.choice([2.0, 4.0, 8.0]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "backward": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + 11)


def _latents(B, H, L, D, dtype, cent, g):
    """(B, L, H, D): runs of neighbouring tokens share one of the centroids `cent` (B, H, 64, D), plus noise."""
    run = max(8, L // 200)
    cid = ((torch.arange(L, device="cuda") // run) * 37) % 64
    out = torch.empty(B, L, H, D, dtype=dtype, device="cuda")
    for b in range(B):
        for h in range(H):
            out[b, :, h] = cent[b, h][cid] + 0.3 * torch.randn(L, D, generator=g, device="cuda")
    return out, cid


def _noise(B, H, L, D, dtype, g):
    out = torch.empty(B, L, H, D, dtype=dtype, device="cuda")
    for b in range(B):
        out[b] = torch.randn(L, H, D, generator=g, device="cuda")
    return out


def _tiles_per_group(case):
    """Valid 128-token tiles of every (batch, head, group): a pattern, so that the work follows from the case."""
    B, H, M, T = case["B"], case["H"], -(-case["L"] // case["rows"]), case["K"] // 128
    if not case["lengths"]:
        return torch.full((B, H, M), T, dtype=torch.int32)
    b, h, m = torch.arange(B).view(B, 1, 1), torch.arange(H).view(1, H, 1), torch.arange(M).view(1, 1, M)
    return (1 + (7 * m + 3 * h + 5 * b) % T).to(torch.int32)


def _indices(B, H, M, L, K, g):
    """Ascending lists of K different tokens: the sinks and the best of random scores that favour whole runs of tokens."""
    run = max(8, L // 200)
    runs = -(-L // run)
    out = torch.empty(B, H, M, K, dtype=torch.int32, device="cuda")
    for b in range(B):
        for h in range(H):
            s = torch.rand(M, L, generator=g, device="cuda")
            s += 0.6 * torch.rand(M, runs, generator=g, device="cuda").repeat_interleave(run, dim=1)[:, :L]
            s[:, :SINKS] = float("inf")
            out[b, h] = s.topk(K, dim=-1).indices.sort(dim=-1).values
    return out


def _positions(case, g):
    """Token positions: the (frame, row, column) grid, or for one axis a run of positions per sequence from a far start."""
    B, L = case["B"], case["L"]
    if case["axes"] == 3:
        t = torch.arange(L, device="cuda")
        return torch.stack([t // 1560, t % 1560 // 40, t % 40], dim=-1)
    start = torch.randint(0, 1 << 20, (B, 1), generator=g, device="cuda")
    return start + torch.arange(L, device="cuda")


def _pairs(case):
    """Rotation pairs of every axis."""
    n = case["rot"] // 2
    if case["axes"] == 1:
        return [n]
    per = case["rot"] // 6
    return [n - 2 * per, per, per]


def prepare(case, seed):
    g = _generator(seed)
    dt, D = DTYPES[case["dtype"]], case["D"]
    if case["kind"] == "rope":
        B, L = case["B"], case["L"]
        q, k = _noise(B, case["Hq"], L, D, dt, g), _noise(B, case["Hk"], L, D, dt, g)
        st = {"case": case, "q": q, "k": k, "positions": _positions(case, g)}
        if own:
            from mcsparse_b200.kernels.flash_mcsa.ops.rotary import RotaryEmbedding
            st["rope"] = RotaryEmbedding(D, rotary_dim=case["rot"], axis_pairs=_pairs(case), layout=case["layout"],
                                         scaling=None if case["scaling"] == "none" else case["scaling"], factor=case["factor"],
                                         original_length=4096)
        return st
    B, H = case["B"], case["H"]
    Lq, Lk = (case["L"], case["L"]) if case["kind"] == "gather" else (case["Lq"], case["Lk"])
    amp = torch.linspace(0.55, 0.85, H, device="cuda").view(1, H, 1, 1) * (128.0 / D) ** 0.25
    cent = amp * torch.randn(B, H, 64, D, generator=g, device="cuda")
    q, cid = _latents(B, H, Lq, D, dt, cent, g)
    k, _ = _latents(B, H, Lk, D, dt, cent, g)
    v, dout = _noise(B, H, Lk, D, dt, g), _noise(B, H, Lq, D, dt, g)
    st = {"case": case, "q": q, "k": k, "v": v, "dout": dout}
    if case["kind"] == "gather":
        M = -(-Lq // case["rows"])
        st["gi"] = _indices(B, H, M, Lk, case["K"], g)
        st["gl"] = _tiles_per_group(case).cuda() if case["lengths"] else None
        st["perm"] = None
        if case["perm"]:
            st["perm"] = torch.stack([torch.argsort(cid + 0.9 * torch.rand(Lq, generator=g, device="cuda")) for _ in range(B * H)])
        st["out"], st["lse"] = _gather_forward(st)
        return st
    # (B, H, L, D) views, as the dense call takes them
    for name in ("q", "k", "v", "dout"):
        st[name] = st[name].transpose(1, 2)
    st["out"], st["lse"] = _dense_forward(st)
    return st


# ------------------------------------------------------------------------------------------------- plain forms
ROWS = 4096                    # query rows whose scores are held at a time


def _dense_forward(st):
    q, k, v = st["q"], st["k"], st["v"]
    B, H, Lq, D = q.shape
    out = torch.empty_like(q)
    lse = torch.empty(B, H, Lq, device=q.device)
    for b in range(B):
        for h in range(H):
            kf, vf = k[b, h].float(), v[b, h].float()
            for r in range(0, Lq, ROWS):
                s = (q[b, h, r:r + ROWS].float() @ kf.t()) * D ** -0.5
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - m)
                z = e.sum(-1, keepdim=True)
                out[b, h, r:r + ROWS] = (e @ vf / z).to(q.dtype)
                lse[b, h, r:r + ROWS] = (m + torch.log(z))[:, 0]
    return out, lse


def _dense_backward(st):
    q, k, v, dout = st["q"], st["k"], st["v"], st["dout"]
    B, H, Lq, D = q.shape
    scale = D ** -0.5
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for b in range(B):
        for h in range(H):
            kf, vf = k[b, h].float(), v[b, h].float()
            dkf, dvf = torch.zeros_like(kf), torch.zeros_like(vf)
            for r in range(0, Lq, ROWS):
                qf, gf = q[b, h, r:r + ROWS].float(), dout[b, h, r:r + ROWS].float()
                s = (qf @ kf.t()) * scale
                p = torch.exp(s - s.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                dvf += p.t() @ gf
                dp = gf @ vf.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[b, h, r:r + ROWS] = (ds @ kf).to(q.dtype)
                dkf += ds.t() @ qf
            dk[b, h], dv[b, h] = dkf.to(k.dtype), dvf.to(v.dtype)
    return dq, dk, dv


def _grouped(x, perm, rows, groups):
    """Rows of x (L, D) in permuted order as (groups, rows, D) in 32 bits, zeros behind the last one."""
    x = x.float() if perm is None else x[perm].float()
    pad = torch.zeros(groups * rows, x.shape[1], device=x.device)
    pad[:x.shape[0]] = x
    return pad.view(groups, rows, -1)


def _gather_forward(st):
    c, q, k, v, gi, gl, perm = st["case"], st["q"], st["k"], st["v"], st["gi"], st["gl"], st["perm"]
    B, L, H, D = q.shape
    M, K = gi.shape[2:]
    out, lse = torch.empty_like(q), torch.empty(B, H, L, device=q.device)
    slot = torch.arange(K, device=q.device) // 128
    for b in range(B):
        for h in range(H):
            pm = None if perm is None else perm[b * H + h]
            idx = gi[b, h].long()
            s = _grouped(q[b, :, h], pm, c["rows"], M) @ k[b, :, h].float()[idx].transpose(1, 2) * D ** -0.5
            if gl is not None:
                s = torch.where(slot < gl[b, h].view(M, 1, 1), s, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - m)
            z = e.sum(-1, keepdim=True)
            o = (e @ v[b, :, h].float()[idx] / z).view(-1, D)[:L].to(q.dtype)
            l = (m + torch.log(z)).view(-1)[:L]
            if pm is None:
                out[b, :, h], lse[b, h] = o, l
            else:
                out[b, pm, h], lse[b, h, pm] = o, l
    return out, lse


def _gather_backward(st):
    c, q, k, v, dout, gi, gl, perm = (st[n] for n in ("case", "q", "k", "v", "dout", "gi", "gl", "perm"))
    B, L, H, D = q.shape
    M, K = gi.shape[2:]
    scale = D ** -0.5
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    slot = torch.arange(K, device=q.device) // 128
    for b in range(B):
        for h in range(H):
            pm = None if perm is None else perm[b * H + h]
            idx = gi[b, h].long()
            kg, vg = k[b, :, h].float()[idx], v[b, :, h].float()[idx]
            qf, gf = _grouped(q[b, :, h], pm, c["rows"], M), _grouped(dout[b, :, h], pm, c["rows"], M)
            s = qf @ kg.transpose(1, 2) * scale
            if gl is not None:
                s = torch.where(slot < gl[b, h].view(M, 1, 1), s, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            dp = gf @ vg.transpose(1, 2)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            dqf = (ds @ kg).view(-1, D)[:L].to(q.dtype)
            if pm is None:
                dq[b, :, h] = dqf
            else:
                dq[b, pm, h] = dqf
            zero = torch.zeros(k.shape[1], D, device=q.device)
            dk[b, :, h] = zero.index_add(0, idx.view(-1), (ds.transpose(1, 2) @ qf).view(-1, D)).to(k.dtype)
            dv[b, :, h] = zero.index_add(0, idx.view(-1), (p.transpose(1, 2) @ gf).view(-1, D)).to(v.dtype)
    return dq, dk, dv


def _frequencies(case):
    """(frequency of every pair, its axis, magnitude) in 64 bits."""
    freq, axis, mag = [], [], 1.0
    for a, n in enumerate(_pairs(case)):
        i = torch.arange(n, dtype=torch.float64)
        f = 10000.0 ** (-i / max(n, 1))
        s = case["factor"]
        if case["scaling"] == "linear":
            f = f / s
        elif case["scaling"] == "ntk":
            f = (10000.0 * s ** (n / (n - 1))) ** (-i / n) if n > 1 else f / s
        elif case["scaling"] == "yarn":
            keep = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
            f = keep * f + (1.0 - keep) * f / s
            mag = 0.1 * math.log(s) + 1.0
        freq.append(f)
        axis += [a] * n
    return torch.cat(freq).cuda(), torch.tensor(axis, device="cuda"), mag


def _rope(st):
    c = st["case"]
    freq, axis, mag = _frequencies(c)
    pos = st["positions"]
    pos = (pos.unsqueeze(-1) if c["axes"] == 1 else pos)[..., axis]
    ang = pos.double() * freq                                # far positions: 32 bits would lose the angle
    if ang.dim() == 2:
        ang = ang.unsqueeze(0)
    cos, sin = (mag * torch.cos(ang)).float().unsqueeze(2), (mag * torch.sin(ang)).float().unsqueeze(2)
    if c["backward"]:
        sin = -sin
    n = c["rot"] // 2
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["layout"] == "interleaved" else (slice(0, n), slice(n, 2 * n))
    res = []
    for x in (st["q"], st["k"]):
        xa, xb = x[..., a].float(), x[..., b].float()
        y = x.float().clone()
        y[..., a] = xa * cos - xb * sin
        y[..., b] = xa * sin + xb * cos
        res.append(y.to(x.dtype))
    return tuple(res)


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return _rope(st) if kind == "rope" else (_gather_backward(st) if kind == "gather" else _dense_backward(st))
    if kind == "rope":
        turn = st["rope"].rotate_backward if st["case"]["backward"] else st["rope"].rotate
        return turn(st["q"], st["k"], positions=st["positions"])
    if kind == "gather":
        from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_backward_func
        return flash_attn_gather_kv_backward_func(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"], st["gi"],
                                                  gather_kv_lengths=st["gl"], perm=st["perm"], group_rows=st["case"]["rows"])
    from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward
    return full_attention_backward(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"])


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    B, D = case["B"], case["D"]
    if case["kind"] == "rope":
        n = B * case["L"] * (case["Hq"] + case["Hk"])
        pos = case["L"] * 3 * 8 if case["axes"] == 3 else B * case["L"] * 8
        return {"bytes": 2 * n * D * es + pos, "flops": 3 * n * case["rot"]}
    H = case["H"]
    if case["kind"] == "dense":
        Lq, Lk = case["Lq"], case["Lk"]
        return {"bytes": B * H * (4 * Lq + 4 * Lk) * D * es + 4 * B * H * Lq, "flops": 10 * B * H * Lq * Lk * D}
    L, rows = case["L"], case["rows"]
    tiles = _tiles_per_group(case)
    left = L - rows * torch.arange(tiles.shape[2])
    columns = int((tiles * left.clamp(max=rows)).sum()) * 128      # (query row, key) pairs
    return {"bytes": B * H * 8 * L * D * es + 4 * B * H * L + 4 * 128 * int(tiles.sum()), "flops": 10 * columns * D}


# ------------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_rope(st):
    c = st["case"]
    freq, axis, mag = _frequencies(c)
    pos = st["positions"].double()
    pos = pos.reshape(1 if c["axes"] == 3 else c["B"], c["L"], 1, c["axes"])
    turn = torch.polar(torch.full_like(freq, mag).expand(pos.shape[0], c["L"], 1, -1).contiguous(), pos[..., axis] * freq)
    if c["backward"]:
        turn = turn.conj()
    n, res = c["rot"] // 2, []
    for x in (st["q"], st["k"]):
        x = x.double()
        head, rest = x[..., :2 * n], x[..., 2 * n:]
        pairs = head.unflatten(-1, (n, 2)) if c["layout"] == "interleaved" else head.unflatten(-1, (2, n)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = y.flatten(-2) if c["layout"] == "interleaved" else y.transpose(-1, -2).flatten(-2)
        res.append(torch.cat([y, rest], dim=-1))
    return tuple(res)


def _gradients(q, k, v, dout, hide=None):
    """Gradients of softmax(q k^T / sqrt(D)) v for the gradient `dout` of its value, by differentiating the definition."""
    with torch.enable_grad():
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        s = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
        if hide is not None:
            s = s.masked_fill(hide, -math.inf)
        return torch.autograd.grad((torch.softmax(s, -1) @ v * dout).sum(), (q, k, v))


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(st)
    q, k, v, dout = (st[n].double() for n in ("q", "k", "v", "dout"))
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if case["kind"] == "dense":
        step = max(1, (1 << 26) // k.shape[2])
        for b in range(q.shape[0]):
            for h in range(q.shape[1]):
                for r in range(0, q.shape[2], step):
                    a, bk, bv = _gradients(q[b, h, r:r + step], k[b, h], v[b, h], dout[b, h, r:r + step])
                    dq[b, h, r:r + step] = a
                    dk[b, h] += bk
                    dv[b, h] += bv
        return dq, dk, dv
    rows, K = case["rows"], case["K"]
    L, M, H = case["L"], st["gi"].shape[2], case["H"]
    for b in range(case["B"]):
        for h in range(H):
            order = torch.arange(L, device=q.device) if st["perm"] is None else st["perm"][b * H + h]
            # rows of every group, the last group's missing ones as row `L` of a padded copy
            member = torch.full((M * rows,), L, device=q.device)
            member[:L] = order
            member = member.view(M, rows)
            zero = torch.zeros(1, q.shape[-1], dtype=q.dtype, device=q.device)
            qp, gp = torch.cat([q[b, :, h], zero]), torch.cat([dout[b, :, h], zero])
            idx = st["gi"][b, h].long()
            hide = None
            if st["gl"] is not None:
                hide = (torch.arange(K, device=q.device) >= 128 * st["gl"][b, h].view(M, 1)).view(M, 1, K)
            step = max(1, (1 << 26) // (rows * K))
            dqp = torch.zeros_like(qp)
            for m in range(0, M, step):
                e = min(M, m + step)
                a, bk, bv = _gradients(qp[member[m:e]], k[b, idx[m:e], h], v[b, idx[m:e], h], gp[member[m:e]],
                                       None if hide is None else hide[m:e])
                dqp.index_copy_(0, member[m:e].reshape(-1), a.reshape(-1, a.shape[-1]))
                flat = idx[m:e].reshape(-1)
                dk[b, :, h].index_add_(0, flat, bk.reshape(-1, bk.shape[-1]))
                dv[b, :, h].index_add_(0, flat, bv.reshape(-1, bv.shape[-1]))
            dq[b, :, h] = dqp[:L]
    return dq, dk, dv
