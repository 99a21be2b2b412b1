"""Cases that time the framework's causal decay attention, group norm with an activation, and residual dropout.

The three make up one causal mixing block on frames, x + dropout(w_o(group_norm_silu(decay_attention(q, k, v)))):

  decay attention   S_t = lambda_h S_(t-1) + k_t v_t^T,  o_t = scale * S_t^T q_t   (one decay lambda_h per head)
  group norm        y = act((x - mean) / sqrt(var + eps) * weight + bias), channels last, statistics for each
                    sample (an utterance's frames, or a single frame) and group of channels
  dropout           y = residual + keep(seeds, position) * x / (1 - p), the keep decisions from a counter-based hash

With `own` false every operator runs in its plain form (elementary torch operations, 32 bits); with `own` true
the framework's entry points are called.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
HEADS, WIDTH = 6, 64  # the encoder's attention: 384 channels as six heads of 64


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    h = {"heads": HEADS, "dk": WIDTH, "dv": WIDTH}
    c = HEADS * WIDTH
    return [
        # one frame of each of four live microphones: nothing but latency
        {"name": "step, 4 streams", "op": "step", "batch": 4, **h, "dtype": "bf16"},
        # one frame of a server's thousand streams, some of them silent: the states' traffic
        {"name": "step, 1000 streams", "op": "step", "batch": 1000, **h, "dtype": "f32"},
        # half a second of audio for each of 24 streams, carried on from the state before
        {"name": "chunk of 50 frames", "op": "prompt", "batch": 24, "frames": 50, **h, "dtype": "bf16", "state": True},
        # one recording of four minutes, and its state for what follows
        {"name": "long recording", "op": "prompt", "batch": 1, "frames": 23999, **h, "dtype": "bf16", "state": True},
        # a padded batch of utterances, offline
        {"name": "utterances, inference", "op": "prompt", "batch": 64, "frames": 400, **h, "dtype": "bf16", "state": False},
        # the training batch, q | k | v from one projection
        {"name": "utterances, training", "op": "train", "batch": 64, "frames": 400, **h, "dtype": "bf16", "packed": True},
        # the same in 32 bits at the small batch
        {"name": "utterances, training f32", "op": "train", "batch": 16, "frames": 400, **h, "dtype": "f32", "packed": False},
        # thirty-second utterances in training: the largest
        {"name": "30 s, training", "op": "train", "batch": 32, "frames": 3000, **h, "dtype": "bf16", "packed": True},
        # every frame's heads normalised behind the attention, inference
        {"name": "head norm", "op": "norm", "batch": 64 * 400, "frames": 0, "channels": c, "groups": HEADS, "act": "silu", "dtype": "bf16", "train": False},
        # utterances normalised over their frames, training batch
        {"name": "utterance norm, training", "op": "norm", "batch": 64, "frames": 400, "channels": c, "groups": 32, "act": "silu", "dtype": "bf16", "train": True},
        # thirty-second utterances in 32 bits, training
        {"name": "30 s norm, training f32", "op": "norm", "batch": 32, "frames": 3000 - 1, "channels": c, "groups": 8, "act": "relu", "dtype": "f32", "train": True},
        # the residual branch's dropout of the training batch, forward and backward
        {"name": "residual dropout", "op": "dropout", "batch": 64, "frames": 400, "channels": c, "p": 0.1, "dtype": "bf16", "residual": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "prompt", "prompt", "train", "train", "norm", "norm", "norm", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("step", "prompt", "train"):
        heads = rng.choice([1, 2, 4, 6, 8, 12])
        dk = rng.choice([32, 64, 64, 128])
        dv = dk if rng.random() < 0.7 else rng.choice([32, 64, 128])
        case = {"op": op, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype}
        if op == "step":
            return {"op": op, "batch": max(1, min(_log(rng, 1, 2000), 4_000_000 * 6 // (heads * dk * dv))), **case}
        frames = _log(rng, 2, 24000 if op == "prompt" else 4000)
        most = max(1, 12_000_000 // (frames * heads * max(dk, dv)))
        batch = min(_log(rng, 1, 96), most)
        if op == "prompt":
            return {**case, "batch": batch, "frames": frames, "state": rng.random() < 0.6}
        return {**case, "batch": batch, "frames": frames, "packed": dk == dv and rng.random() < 0.5}
    channels = rng.choice([80, 96, 128, 192, 256, 384, 384, 512, 640, 1000])
    if op == "norm":
        groups = rng.choice([g for g in (1, 2, 4, 5, 6, 8, 10, 16, 20, 32) if channels % g == 0])
        frames = 0 if rng.random() < 0.4 else _log(rng, 2, 4000)
        rows = _log(rng, 1, 30000) if frames == 0 else max(1, min(_log(rng, 1, 96), 30_000_000 // (frames * channels)))
        return {"op": op, "batch": rows, "frames": frames, "channels": channels, "groups": groups,
                "act": rng.choice(["none", "relu", "silu"]), "dtype": dtype, "train": rng.random() < 0.6}
    frames = _log(rng, 1, 4000)
    batch = max(1, min(_log(rng, 1, 96), 25_000_000 // (frames * channels)))
    return {"op": op, "batch": batch, "frames": frames, "channels": channels + rng.choice([0, 0, 1, 2]),
            "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "dtype": dtype, "residual": rng.choice(["none", "bf16", "f32"])}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _lengths(batch, frames, seed):
    """Frames of each utterance of a padded batch: the longest fills it, the others spread down to a tenth."""
    g = torch.Generator().manual_seed(int(seed) + 17)
    n = torch.randint(max(1, frames // 10), frames + 1, (batch,), generator=g, dtype=torch.int32)
    n[int(torch.randint(0, batch, (1,), generator=g))] = frames
    return n.cuda()


def prepare(case, seed):
    g = _generator(seed)
    dt = DT[case["dtype"]]
    op, B = case["op"], case["batch"]
    s = {"case": case}

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    if op in ("step", "prompt", "train"):
        H, dk, dv = case["heads"], case["dk"], case["dv"]
        # slow decays, each head twice as slow as the one before, a little off for each seed
        base = 5.0 + torch.rand(1, generator=g, device="cuda", dtype=torch.float64)
        h = torch.arange(H, device="cuda", dtype=torch.float64) % 8
        s["log_decay"] = torch.log1p(-torch.exp2(-base - h)).float()
        if op == "step":
            s["q"], s["k"], s["v"] = normal(B, H * dk), normal(B, H * dk), normal(B, H * dv)
            s["state"] = normal(B, H, dk, dv, dtype=torch.float32) * 4
            s["active"] = (torch.rand(B, generator=g, device="cuda") < 0.9).to(torch.int32)
            return s
        T = case["frames"]
        s["lengths"] = _lengths(B, T, seed)
        if case.get("packed"):
            s["qkv"] = normal(B, T, 3 * H * dk)
        else:
            s["q"], s["k"], s["v"] = normal(B, T, H * dk), normal(B, T, H * dk), normal(B, T, H * dv)
        if op == "train":
            s["dout"] = normal(B, T, H * dv)
            for name in ("qkv", "q", "k", "v"):
                if name in s:
                    s[name].requires_grad_(True)
        elif case["state"]:
            s["state"] = normal(B, H, dk, dv, dtype=torch.float32) * 4
        return s
    C, T = case["channels"], case["frames"]
    shape = (B, T, C) if T else (B, C)
    if op == "norm":
        spread = 0.5 + torch.rand(C, generator=g, device="cuda")
        middle = torch.randn(C, generator=g, device="cuda")
        s["x"] = (torch.randn(*shape, generator=g, device="cuda") * spread + middle).to(dt)
        s["weight"] = 1 + 0.2 * torch.randn(C, generator=g, device="cuda")
        s["bias"] = 0.2 * torch.randn(C, generator=g, device="cuda")
        s["lengths"] = _lengths(B, T, seed) if T else None
        if case["train"]:
            s["dout"] = normal(*shape)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
        return s
    s["x"] = normal(*shape).requires_grad_(True)
    s["residual"] = None if case["residual"] == "none" else normal(*shape, dtype=DT[case["residual"]])
    out = dt if s["residual"] is None else torch.promote_types(dt, s["residual"].dtype)
    s["dout"] = normal(*shape, dtype=out)
    s["seeds"] = (int(seed) & 0x7FFFFFFF, (int(seed) * 2654435761 + 12345) & 0xFFFFFFFF)
    return s


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B = case["batch"]
    if case["op"] in ("step", "prompt", "train"):
        H, dk, dv = case["heads"], case["dk"], case["dv"]
        n = B * case.get("frames", 1) * H
        state = B * H * dk * dv * 4
        tensors = n * (2 * dk + 2 * dv) * e  # q, k, v in, the output out
        if case["op"] == "step":
            return {"bytes": tensors + 2 * state, "flops": 4 * n * dk * dv}
        if case["op"] == "prompt":
            return {"bytes": tensors + (2 * state if case["state"] else 0), "flops": 4 * n * dk * dv}
        return {"bytes": tensors + n * (2 * dk + 2 * dv) * e, "flops": 14 * n * dk * dv}
    n = B * max(1, case["frames"]) * case["channels"]
    if case["op"] == "norm":
        return {"bytes": (4 if case["train"] else 2) * n * e, "flops": (24 if case["train"] else 10) * n}
    r = {"none": 0, "bf16": 2, "f32": 4}[case["residual"]]
    out = max(e, r)
    return {"bytes": n * (e + r + out) + n * (out + e), "flops": 6 * n}


# ------------------------------------------------------------------------------------------------ plain forms

_CHUNK = 128  # frames whose scores the plain form holds as one square


def _plain_decay(q, k, v, log_decay, heads, lengths, state):
    """(output, state after each row's last frame): squares of scores inside chunks of frames, the chunks' states
    joined by one product with the powers of the decays.  q, k [B, T, H dk], v [B, T, H dv], all float32."""
    B, T, _ = q.shape
    dk, dv = q.shape[2] // heads, v.shape[2] // heads
    C = min(_CHUNK, T)
    n = -(-T // C)
    a = log_decay.double()
    at = torch.arange(n * C, device=q.device)
    inside = at[None, :] < lengths[:, None]  # [B, n C]

    def split(t, d):
        t = torch.nn.functional.pad(t, (0, 0, 0, n * C - T))
        t = torch.where(inside[:, :, None], t, torch.zeros((), device=t.device))
        return t.reshape(B, n, C, heads, d).permute(0, 3, 1, 2, 4)  # [B, H, n, C, d]

    q, k, v = split(q, dk) * dk ** -0.5, split(k, dk), split(v, dv)
    i = torch.arange(C, device=q.device)
    gap = i[:, None] - i[None, :]
    square = torch.where(gap >= 0, torch.exp(a[:, None, None] * gap.clamp(min=0)), 0.0).float()  # [H, C, C]
    out = ((q @ k.transpose(-1, -2)) * square[None, :, None]) @ v
    to_end = torch.exp(a[:, None] * (C - 1 - i)).float()
    local = (k * to_end[None, :, None, :, None]).transpose(-1, -2) @ v  # what each chunk adds: [B, H, n, dk, dv]
    c = torch.arange(n, device=q.device)
    gap = c[:, None] - 1 - c[None, :]
    across = torch.where(gap >= 0, torch.exp(a[:, None, None] * C * gap.clamp(min=0)), 0.0).float()  # [H, n, n]
    before = (across[None] @ local.reshape(B, heads, n, dk * dv)).reshape(B, heads, n, dk, dv)
    if state is not None:
        before = before + torch.exp(a[:, None] * C * c).float()[None, :, :, None, None] * state[:, :, None]
    from_start = torch.exp(a[:, None] * (i + 1)).float()
    out = out + from_start[None, :, None, :, None] * (q @ before)
    out = out.permute(0, 2, 3, 1, 4).reshape(B, n * C, heads * dv)[:, :T]
    if state is None:
        return out, None
    left = lengths[:, None, None].double() - 1 - at  # [B, 1, n C]
    weight = torch.where(left >= 0, torch.exp(a[None, :, None] * left.clamp(min=0)), 0.0).float()
    k, v = k.reshape(B, heads, n * C, dk), v.reshape(B, heads, n * C, dv)
    new = (k * weight[..., None]).transpose(-1, -2) @ v
    return out, new + torch.exp(a[None, :] * lengths[:, None].double()).float()[:, :, None, None] * state


def _plain_norm(x, weight, bias, groups, act, lengths):
    x3 = x.float() if x.dim() == 3 else x.float()[:, None]
    B, T, C = x3.shape
    xg = x3.reshape(B, T, groups, C // groups)
    if lengths is None:
        inside = torch.ones(B, T, 1, 1, dtype=torch.bool, device=x.device)
        count = torch.full((B, 1, 1, 1), float(T * (C // groups)), device=x.device)
    else:
        inside = (torch.arange(T, device=x.device)[None, :] < lengths[:, None])[:, :, None, None]
        count = (lengths.float() * (C // groups)).clamp(min=1)[:, None, None, None]
    zero = torch.zeros((), device=x.device)
    mean = torch.where(inside, xg, zero).sum(dim=(1, 3), keepdim=True) / count
    centred = torch.where(inside, xg - mean, zero)
    var = (centred * centred).sum(dim=(1, 3), keepdim=True) / count
    y = (centred * torch.rsqrt(var + 1e-5)).reshape(B, T, C) * weight + bias
    if act == "relu":
        y = torch.relu(y)
    elif act == "silu":
        y = y * torch.sigmoid(y)
    y = torch.where(inside.reshape(B, T, 1), y, zero)
    return y.reshape(x.shape).to(x.dtype)


def _plain_keep(shape, p, seeds, device):
    """The keep decisions: columns 2c and 2c + 1 of a row share one 32-bit hash of the pair's index and the seeds
    (MurmurHash3's finaliser) and read its low and high half."""
    C = shape[-1]
    rows = math.prod(shape[:-1])
    low = 0xFFFFFFFF
    pairs = (C + 1) // 2
    col = torch.arange(C, device=device)
    g = torch.arange(rows, device=device)[:, None] * pairs
    mixed = seeds[0] ^ ((((g >> 32) + seeds[1]) * 0x9E3779B1) & low)
    h = (((g & low) + (col >> 1)) & low) ^ mixed
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & low
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & low
    h = h ^ (h >> 16)
    field = (h >> (16 * (col & 1))) & 0xFFFF
    return (field >= min(max(int(p * 65536 + 0.5), 1), 65535)).reshape(shape)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "step":
        H, dk, dv = case["heads"], case["dk"], case["dv"]
        B = case["batch"]
        q, k, v = s["q"].float().view(B, H, dk), s["k"].float().view(B, H, dk), s["v"].float().view(B, H, dv)
        live = (s["active"] > 0)[:, None, None, None]
        new = torch.exp(s["log_decay"])[None, :, None, None] * s["state"] + k[..., None] * v[:, :, None, :]
        out = (q[:, :, None, :] * dk ** -0.5) @ new
        s["state"].copy_(torch.where(live, new, s["state"]))
        out = torch.where(live, out, torch.zeros((), device=out.device))
        return out.reshape(B, H * dv).to(s["q"].dtype), s["state"]
    if op == "prompt":
        out, state = _plain_decay(s["q"].float(), s["k"].float(), s["v"].float(), s["log_decay"], case["heads"],
                                  s["lengths"], s.get("state"))
        out = out.to(s["q"].dtype)
        if state is None:
            return out
        s["state"].copy_(state)
        return out, s["state"]
    if op == "train":
        if case["packed"]:
            q, k, v = s["qkv"].float().chunk(3, dim=-1)
            leaves = (s["qkv"],)
        else:
            q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
            leaves = (s["q"], s["k"], s["v"])
        out, _ = _plain_decay(q, k, v, s["log_decay"], case["heads"], s["lengths"], None)
        out = out.to(s["dout"].dtype)
        return (out.detach(), *torch.autograd.grad(out, leaves, s["dout"]))
    if op == "norm":
        y = _plain_norm(s["x"], s["weight"], s["bias"], case["groups"], case["act"], s["lengths"])
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dout"]))
    keep = _plain_keep(s["x"].shape, case["p"], s["seeds"], s["x"].device)
    y = torch.where(keep, s["x"].float() / (1.0 - case["p"]), torch.zeros((), device=keep.device))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(s["dout"].dtype)
    return (y.detach(), *torch.autograd.grad(y, (s["x"],), s["dout"]))


# ------------------------------------------------------------------------------------------------ the framework

def _run_own(s):
    case = s["case"]
    op = case["op"]
    if op in ("step", "prompt", "train"):
        from asr_amd import decay

        if op == "step":
            out = decay.decay_attention_step(s["q"], s["k"], s["v"], case["heads"], s["log_decay"], s["state"], s["active"])
            return out, s["state"]
        if op == "prompt":
            out = decay.decay_attention(s["q"], s["k"], s["v"], case["heads"], s["log_decay"], s["lengths"], s.get("state"))
            return (out, s["state"]) if "state" in s else out
        if case["packed"]:
            out = decay.decay_attention_train_packed(s["qkv"], case["heads"], s["log_decay"], s["lengths"])
            leaves = (s["qkv"],)
        else:
            out = decay.decay_attention_train(s["q"], s["k"], s["v"], case["heads"], s["log_decay"], s["lengths"])
            leaves = (s["q"], s["k"], s["v"])
        return (out.detach(), *torch.autograd.grad(out, leaves, s["dout"]))
    if op == "norm":
        from asr_amd import groupnorm

        act = None if case["act"] == "none" else case["act"]
        if not case["train"]:
            return groupnorm.group_norm(s["x"], case["groups"], s["weight"], s["bias"], 1e-5, act, s["lengths"])
        y = groupnorm.group_norm_train(s["x"], case["groups"], s["weight"], s["bias"], 1e-5, act, s["lengths"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dout"]))
    from asr_amd import dropout

    y = dropout.dropout_add(s["x"], s["residual"], case["p"], s["seeds"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"],), s["dout"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    def decay(s, case, q, k, v):
        """Frame by frame from the recurrence; with "dout" also the gradients, frame by frame backwards."""
        H, dk, dv = case["heads"], case["dk"], case["dv"]
        B, T, _ = q.shape
        lam = torch.exp(s["log_decay"].double())[None, :, None, None]
        q, k, v = q.double().view(B, T, H, dk) * dk ** -0.5, k.double().view(B, T, H, dk), v.double().view(B, T, H, dv)
        S = s["state"].double().clone() if "state" in s else torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device)
        live = (torch.arange(T, device=q.device)[:, None] < s["lengths"][None, :])[:, :, None, None, None]  # [T, B, 1, 1, 1]
        out = torch.zeros(B, T, H, dv, dtype=torch.float64, device=q.device)
        train = "dout" in s
        if train:
            do = s["dout"].double().view(B, T, H, dv)
            dq, dkey, dval = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        for t in range(T):
            S = torch.where(live[t], lam * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
            out[:, t] = torch.where(live[t][..., 0], (q[:, t, :, :, None] * S).sum(2), 0.0)
            if train:
                dq[:, t] = torch.where(live[t][..., 0], (S * do[:, t, :, None, :]).sum(3) * dk ** -0.5, 0.0)
        if not train:
            return out.view(B, T, H * dv), S
        G = torch.zeros_like(S)
        for t in range(T - 1, -1, -1):
            G = torch.where(live[t], lam * G + q[:, t, :, :, None] * do[:, t, :, None, :], G)
            dkey[:, t] = torch.where(live[t][..., 0], (G * v[:, t, :, None, :]).sum(3), 0.0)
            dval[:, t] = torch.where(live[t][..., 0], (G * k[:, t, :, :, None]).sum(2), 0.0)
        return out.view(B, T, H * dv), dq.view(B, T, H * dk), dkey.view(B, T, H * dk), dval.view(B, T, H * dv)

    def norm(s, case):
        """Sample by sample, and the gradients from their formulas."""
        train = "dout" in s
        x = s["x"].detach().double()
        C, G = case["channels"], case["groups"]
        w, b = s["weight"].detach().double(), s["bias"].detach().double()
        frames = case["frames"]
        samples = [(i, int(n)) for i, n in enumerate(s["lengths"].tolist())] if frames else [(slice(None), 0)]
        y, dx = torch.zeros_like(x), torch.zeros_like(x)
        dw, db = torch.zeros_like(w), torch.zeros_like(b)
        for i, n in samples:
            # single frames are all done at once: a frame is a row of [rows, G, C / G]; an utterance is [1, frames, G, C / G]
            at = (i, slice(0, n)) if frames else (i,)
            part = x[at].reshape(-1, 1, G, C // G) if not frames else x[at].reshape(1, n, G, C // G)
            mean = part.mean(dim=(1, 3), keepdim=True)
            std = torch.sqrt(((part - mean) ** 2).mean(dim=(1, 3), keepdim=True) + 1e-5)
            hat = (part - mean) / std
            W = w.view(G, C // G)
            z = hat * W + b.view(G, C // G)
            sig = 1 / (1 + torch.exp(-z))
            f = {"none": z, "relu": z.clamp(min=0), "silu": z * sig}[case["act"]]
            y[at] = f.reshape(x[at].shape)
            if train:
                slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": sig * (1 + z * (1 - sig))}[case["act"]]
                dz = s["dout"][at].double().reshape(part.shape) * slope
                dw += (dz * hat).sum(dim=(0, 1)).reshape(C)
                db += dz.sum(dim=(0, 1)).reshape(C)
                gy = dz * W
                d = (gy - gy.mean(dim=(1, 3), keepdim=True) - hat * (gy * hat).mean(dim=(1, 3), keepdim=True)) / std
                dx[at] = d.reshape(x[at].shape)
        return (y, dx, dw, db) if train else y

    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "step":
            B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
            one = dict(s, lengths=s["active"])
            out, S = decay(one, case, s["q"].view(B, 1, -1), s["k"].view(B, 1, -1), s["v"].view(B, 1, -1))
            return out.view(B, H * dv), S
        if case["op"] == "prompt":
            out, S = decay(s, case, s["q"], s["k"], s["v"])
            return (out, S) if case["state"] else out
        if case["op"] == "train":
            q, k, v = s["qkv"].chunk(3, dim=-1) if case["packed"] else (s["q"], s["k"], s["v"])
            got = decay(s, case, *(t.contiguous() for t in (q, k, v)))
            return (got[0], torch.cat(got[1:], dim=-1)) if case["packed"] else got
        if case["op"] == "norm":
            return norm(s, case)
        # dropout: the decisions in 32-bit unsigned arithmetic of numpy, row by row of pairs
        import numpy as np

        C = case["channels"]
        rows = s["x"].numel() // C
        pairs = (C + 1) // 2
        first = np.arange(rows, dtype=np.uint64) * np.uint64(pairs)
        with np.errstate(over="ignore"):
            high = (first >> np.uint64(32)).astype(np.uint32) + np.uint32(s["seeds"][1])
            h = first.astype(np.uint32)[:, None] + np.arange(pairs, dtype=np.uint32)[None, :]
            h ^= (np.uint32(s["seeds"][0]) ^ (high * np.uint32(0x9E3779B1)))[:, None]
            for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
                h ^= h >> np.uint32(shift)
                h *= np.uint32(factor)
            h ^= h >> np.uint32(16)
        least = min(max(int(case["p"] * 65536 + 0.5), 1), 65535)
        keep = np.stack([(h & np.uint32(0xFFFF)) >= least, (h >> np.uint32(16)) >= least], axis=2).reshape(rows, 2 * pairs)[:, :C]
        scale = torch.from_numpy(keep.copy()).cuda().double().view(s["x"].shape) / (1 - case["p"])
        y = s["x"].detach().double() * scale
        return (y if s["residual"] is None else y + s["residual"].double()), s["dout"].double() * scale
