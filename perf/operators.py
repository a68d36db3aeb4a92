"""The state-space operators and the gradient clip as they are timed: cases, inputs, plain forms and 64-bit definitions.

`own = False` computes each operator from elementary torch operations, `own = True` calls the framework's kernels."""
import math

import torch

own = False
CHUNK = 64  # tokens per chunk of the plain scan
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one stream separated online: a frame's 192 channels (two 64-channel directions and their B, C) through the convolution
        {"name": "conv_step_one_stream", "op": "conv_step", "B": 1, "D": 192, "K": 4, "type": "f32"},
        # a long recording as one prompt: 32 heads of 64 channels plus B and C of 128
        {"name": "conv_prompt_long", "op": "conv", "B": 1, "L": 32768, "D": 2304, "K": 4, "type": "bf16", "ragged": False},
        # training on the time axis of the dual path: 32 utterances x 64 bands, 2 s
        {"name": "conv_train_dual_path", "op": "conv_train", "B": 2048, "L": 125, "D": 192, "K": 4, "type": "f32", "ragged": False},
        # a padded batch of three utterances with an odd channel count
        {"name": "conv_train_odd", "op": "conv_train", "B": 3, "L": 1999, "D": 333, "K": 3, "type": "bf16", "ragged": True},
        # one stream separated online: one frame through the recurrence
        {"name": "scan_step_one_stream", "op": "scan_step", "B": 1, "H": 4, "P": 32, "G": 1, "N": 32, "type": "f32"},
        # 256 streams served together
        {"name": "scan_step_batch", "op": "scan_step", "B": 256, "H": 32, "P": 64, "G": 1, "N": 128, "type": "bf16"},
        # a padded batch of seven prompts, sizes that fill no tile
        {"name": "scan_prompt_ragged", "op": "scan", "B": 7, "L": 501, "H": 6, "P": 48, "G": 2, "N": 40, "type": "f32", "ragged": True},
        # a long recording as one prompt, the state kept for the frames that follow
        {"name": "scan_prompt_long", "op": "scan", "B": 1, "L": 32768, "H": 32, "P": 64, "G": 1, "N": 128, "type": "bf16", "ragged": False},
        # training on the time axis of the dual path, fp32 as the framework trains
        {"name": "scan_train_dual_path", "op": "scan_train", "B": 2048, "L": 125, "H": 4, "P": 32, "G": 1, "N": 32, "type": "f32", "ragged": False},
        # training on long sequences in bf16
        {"name": "scan_train_long", "op": "scan_train", "B": 8, "L": 2048, "H": 32, "P": 64, "G": 1, "N": 128, "type": "bf16", "ragged": False},
        # RTFS-Net's 403 parameter tensors, 740,210 numbers
        {"name": "clip_rtfs_net", "op": "clip", "count": 403, "total": 740210, "type": "f32", "norm": 2.0},
        # the gradients of a large model in bf16
        {"name": "clip_large", "op": "clip", "count": 291, "total": 300_000_000, "type": "bf16", "norm": 2.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["conv_step", "conv", "conv_train", "scan_step", "scan", "scan_train", "scan", "scan_train", "clip"])
    t = rng.choice(["f32", "bf16"])
    if op == "clip":
        total = _spread(rng, 1000, 200_000_000)
        return {"op": op, "count": min(_spread(rng, 1, 600), total // 4), "total": total, "type": t, "norm": rng.choice([2.0, 2.0, math.inf])}
    if op == "conv_step":
        return {"op": op, "B": _spread(rng, 1, 512), "D": _spread(rng, 16, 8192), "K": rng.choice([2, 3, 4, 5]), "type": t}
    if op in ("conv", "conv_train"):
        D, most = _spread(rng, 16, 4096), 30_000_000
        L = _spread(rng, 1, min(32768, most // D))
        return {"op": op, "B": _spread(rng, 1, max(1, min(2048, most // (D * L)))), "L": L, "D": D, "K": rng.choice([2, 3, 4, 5]), "type": t,
                "ragged": rng.random() < 0.4}
    P, N = _spread(rng, 8, 128), _spread(rng, 8, 128)
    G = rng.choice([1, 1, 2, 4])
    H = G * _spread(rng, 1, 32 // G)
    if op == "scan_step":
        return {"op": op, "B": _spread(rng, 1, max(1, min(512, 67_000_000 // (H * P * N)))), "H": H, "P": P, "G": G, "N": N, "type": t}
    # bounded by the work (tokens x H x P x N), by the plain form's chunk states and by its score matrices
    tokens = min(262_144, 3_000_000_000 // (H * P * max(N, 32)), 40_000_000 // (H * max(P, N)))
    L = _spread(rng, 1, min(tokens, 32768 if op == "scan" else 4096))
    return {"op": op, "B": _spread(rng, 1, max(1, min(2048, tokens // (L + CHUNK)))), "L": L, "H": H, "P": P, "G": G, "N": N, "type": t,
            "ragged": rng.random() < 0.4}


def _lengths(case, rnd):
    """rows of a padded batch: the first is full, the others end anywhere from the first token on (an empty one among them where there are four)"""
    if not case.get("ragged"):
        return None
    n = torch.randint(1, case["L"] + 1, (case["B"],), generator=rnd, device="cuda", dtype=torch.int32)
    n[0] = case["L"]
    if case["B"] >= 4:
        n[-1] = 0
    return n


def prepare(case, seed):
    rnd = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, op = TYPES[case["type"]], case["op"]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=rnd, device="cuda") * scale).to(dtype)

    s = {"op": op, "case": dict(case)}
    if op == "clip":
        # the tensors are views of one flat buffer, as data-parallel training keeps its gradients; their sizes differ as a model's do
        count, total = case["count"], case["total"]
        share = torch.rand(count, generator=rnd, device="cuda").mul(4).exp().double().cpu()
        sizes = (share / share.sum() * (total - count)).long() + 1
        sizes[0] += total - int(sizes.sum())
        flat = normal(total, scale=0.02, dtype=kind)
        s["flat"], s["params"] = flat, []
        for g in flat.split(sizes.tolist()):
            p = torch.nn.Parameter(g.detach())  # the weights' values are not read
            p.grad = g
            s["params"].append(p)
        # a first pass scales the gradients to the bound (where they are above it); a further pass on them does the same work with a factor next to 1
        s["max_norm"], s["norm"] = 5.0 if case["norm"] == 2.0 else 0.01, case["norm"]
        return s
    B = case["B"]
    if op.startswith("conv"):
        D, K = case["D"], case["K"]
        s["weight"], s["bias"] = normal(D, K, scale=K ** -0.5), normal(D, scale=0.1)
        s["state"] = normal(B, K - 1, D, dtype=kind)
        if op == "conv_step":
            s["x"] = normal(B, D, dtype=kind)
            return s
        L = case["L"]
        s["lengths"] = _lengths(case, rnd)
        if op == "conv":
            s["x"] = normal(B, L, D + 64, dtype=kind)[..., 32:32 + D]  # a slice of the projection's output
        else:
            s["x"], s["dy"] = normal(B, L, D, dtype=kind), normal(B, L, D, dtype=kind)
        return s
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    step = torch.rand(H, generator=rnd, device="cuda").mul(math.log(100.0)).exp().mul(1e-3)  # step sizes 1e-3 ... 1e-1
    s["dt_bias"] = step.expm1().log()
    s["A"] = -(1 + 15 * torch.rand(H, generator=rnd, device="cuda"))
    s["D"] = 1 + normal(H, scale=0.1)
    s["state"] = normal(B, H, P, N, scale=0.3)
    if op == "scan_step":
        s["x"], s["dt"] = normal(B, H, P, dtype=kind), normal(B, H, scale=0.5, dtype=kind)
        s["B"], s["C"] = normal(B, G, N, dtype=kind), normal(B, G, N, dtype=kind)
        return s
    L = case["L"]
    s["lengths"] = _lengths(case, rnd)
    if op == "scan":  # x, B and C are slices of the convolution's output, dt one of the projection's
        both = normal(B, L, H * P + 2 * G * N, dtype=kind)
        x, b, c = both.split([H * P, G * N, G * N], -1)
        s["x"], s["B"], s["C"] = x.unflatten(-1, (H, P)), b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))
        s["dt"] = normal(B, L, H + 8, scale=0.5, dtype=kind)[..., :H]
    else:
        s["x"], s["dt"] = normal(B, L, H, P, dtype=kind), normal(B, L, H, scale=0.5, dtype=torch.float32)
        s["B"], s["C"] = normal(B, L, G, N, dtype=kind), normal(B, L, G, N, dtype=kind)
        s["dy"], s["dstate"] = normal(B, L, H, P, dtype=kind), normal(B, H, P, N, scale=0.1)
    return s


def run(state):
    op = state["op"]
    if op == "clip":
        return {"norm": _clip(state), "grads": state["flat"]}
    if op == "conv_step":
        y = _conv_step(state)
        return {"y": y, "state": state["state"]}
    if op == "scan_step":
        y = _scan_step(state)
        return {"y": y, "state": state["state"]}
    conv = op.startswith("conv")
    call = _conv if conv else _scan
    if not op.endswith("train"):
        with torch.no_grad():
            y, last = call(state)
        return {"y": y, "state": last}
    names = ("x", "weight", "bias", "state") if conv else ("x", "dt", "A", "B", "C", "D", "dt_bias", "state")
    leaves = {k: state[k].detach().requires_grad_() for k in names}
    y, last = call({**state, **leaves})
    outs, given = ([y], [state["dy"]]) if conv else ([y, last], [state["dy"], state["dstate"]])
    grads = torch.autograd.grad(outs, list(leaves.values()), given)
    return {"y": y.detach(), "last": last.detach(), **{"d_" + k: g for k, g in zip(names, grads)}}


def _clip(s):
    if own:
        from rtfs_net_amd.optim import clip_grad_norm_

        return clip_grad_norm_(s["params"], s["max_norm"], s["norm"])
    grads = [p.grad for p in s["params"]]
    if s["norm"] == math.inf:
        norm = torch.stack([g.abs().max() for g in grads]).max().float()
    else:
        norm = torch.stack(torch._foreach_norm(grads, 2, dtype=torch.float32)).double().square().sum().sqrt().float()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if grads[0].dtype == torch.float32:
        torch._foreach_mul_(grads, coef)
    else:
        [g.copy_(g.float().mul_(coef)) for g in grads]
    return norm


def _conv(s):
    if own:
        from rtfs_net_amd.ssm import causal_conv

        return causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"], return_state=True)
    x, K, n = s["x"].float(), s["weight"].shape[1], s["lengths"]
    L = x.shape[1]
    if n is not None:
        keep = (torch.arange(L, device=x.device) < n[:, None])[..., None]
        x = torch.where(keep, x, 0)
    both = torch.cat([s["state"].float(), x], 1)
    pre = (both.unfold(1, K, 1) * s["weight"]).sum(-1) + s["bias"]
    y = pre * torch.sigmoid(pre)
    if n is None:
        last = both[:, L:]
    else:
        y = torch.where(keep, y, 0)
        at = n[:, None].long() + torch.arange(K - 1, device=x.device)
        last = both.gather(1, at[..., None].expand(-1, -1, x.shape[2]))
    return y.to(s["x"].dtype), last.to(s["x"].dtype)


def _conv_step(s):
    if own:
        from rtfs_net_amd.ssm import causal_conv_step

        return causal_conv_step(s["x"], s["state"], s["weight"], s["bias"])
    both = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = (both.float() * s["weight"].t()).sum(1) + s["bias"]
    s["state"].copy_(both[:, 1:])
    return (pre * torch.sigmoid(pre)).to(s["x"].dtype)


def _scan_step(s):
    if own:
        from rtfs_net_amd.ssm import selective_scan_step

        return selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], s["D"], dt_bias=s["dt_bias"], softplus=True)
    x, each = s["x"].float(), s["x"].shape[1] // s["B"].shape[1]
    dt = torch.logaddexp(s["dt"].float() + s["dt_bias"], torch.zeros((), device=x.device))
    b, c = (s[k].float().repeat_interleave(each, 1) for k in "BC")
    new = s["state"] * (dt * s["A"]).exp()[..., None, None] + (dt[..., None] * x)[..., None] * b[:, :, None]
    s["state"].copy_(new)
    y = (new * c[:, :, None]).sum(-1) + s["D"][:, None] * x
    return y.to(s["x"].dtype)


def _scan(s):
    if own:
        from rtfs_net_amd.ssm import selective_scan

        return selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], dt_bias=s["dt_bias"], softplus=True, state=s["state"],
                              lengths=s["lengths"], return_state=True)
    x, b, c, n = s["x"].float(), s["B"].float(), s["C"].float(), s["lengths"]
    rows, L, H, P = x.shape
    G, N = b.shape[2:]
    dt = torch.logaddexp(s["dt"].float() + s["dt_bias"], torch.zeros((), device=x.device))
    if n is not None:
        keep = torch.arange(L, device=x.device) < n[:, None]
        dt = torch.where(keep[..., None], dt, 0)
    Q = min(CHUNK, L)
    Z = -(-L // Q)

    def chunks(v):  # [rows, L, heads, ...] -> [rows, Z, heads, Q, ...]
        v = torch.cat([v, v.new_zeros(rows, Z * Q - L, *v.shape[2:])], 1) if Z * Q > L else v
        return v.unflatten(1, (Z, Q)).transpose(2, 3)

    each = H // G
    xc, dc = chunks(x), chunks(dt)
    bc, cc = chunks(b), chunks(c)
    sums = (dc.double() * s["A"].double()[:, None]).cumsum(-1)  # log decay up to each token of its chunk
    upper = torch.ones(Q, Q, dtype=torch.bool, device=x.device).triu(1)
    decay = (sums[..., :, None] - sums[..., None, :]).float().masked_fill(upper, -math.inf).exp()
    xd = xc * dc[..., None]
    y = ((cc @ bc.transpose(-1, -2)).repeat_interleave(each, 2) * decay) @ xd
    to_end = (sums[..., -1:] - sums).float().exp()
    ends = (xd * to_end[..., None]).transpose(-1, -2) @ bc.repeat_interleave(each, 2)  # [rows, Z, H, P, N], the chunk's own part of its last state
    whole = torch.cat([sums.new_zeros(rows, H, 1), sums[..., -1].transpose(1, 2).cumsum(-1)], -1)  # log decay up to each chunk's start
    later = torch.ones(Z + 1, Z + 1, dtype=torch.bool, device=x.device).triu(1)
    between = (whole[..., :, None] - whole[..., None, :]).float().masked_fill(later, -math.inf).exp()
    parts = torch.cat([s["state"][:, None], ends], 1).transpose(1, 2).flatten(3)
    starts = (between @ parts).unflatten(-1, (P, N))  # [rows, H, Z + 1, P, N]
    from_start = cc.repeat_interleave(each, 2) @ starts[:, :, :Z].permute(0, 2, 1, 4, 3)
    y = y + from_start * sums.float().exp()[..., None]
    y = y.transpose(2, 3).flatten(1, 2)[:, :L] + s["D"][:, None] * x
    if n is not None:
        y = torch.where(keep[..., None, None], y, 0)
    return y.to(s["x"].dtype), starts[:, :, Z]


def work(case):
    op = case["op"]
    size = 4 if case["type"] == "f32" else 2
    if op == "clip":
        return {"bytes": 3 * case["total"] * size, "flops": 3 * case["total"]}
    B = case["B"]
    if op.startswith("conv"):
        D, K = case["D"], case["K"]
        if op == "conv_step":
            return {"bytes": B * D * size * (2 + 2 * (K - 1)) + 4 * D * (K + 1), "flops": B * D * (2 * K + 5)}
        n = B * case["L"] * D
        return {"bytes": n * size * (2 if op == "conv" else 5), "flops": n * (2 * K + 5) * (1 if op == "conv" else 4)}
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    if op == "scan_step":
        return {"bytes": B * H * P * N * 8 + B * (H * P * 2 + H + 2 * G * N) * size, "flops": B * H * P * N * 5}
    n = B * case["L"]
    if op == "scan":
        return {"bytes": n * (2 * H * P + 2 * G * N + H) * size + B * H * P * N * 8, "flops": n * H * P * N * 5}
    # forward: x, B, C, dt in, y out; backward: those and dy in, dx, dB, dC, ddt out
    return {"bytes": n * (5 * H * P + 6 * G * N) * size + n * 3 * H * 4 + B * H * P * N * 16, "flops": n * H * P * N * 14}


# ---- the definitions, token by token in 64 bits ----------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "clip":
        g = s["flat"].double()
        norm = g.abs().max() if s["norm"] == math.inf else torch.linalg.vector_norm(g)
        return {"norm": norm, "grads": g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
    v = {k: t.double() for k, t in s.items() if torch.is_tensor(t) and k != "lengths"}
    if op.startswith("conv"):
        return _exact_conv(op, v, s.get("lengths"))
    return _exact_scan(op, v, s.get("lengths"))


def _exact_conv(op, v, lengths):
    w, bias, x, first = v["weight"], v["bias"], v["x"], v["state"]
    K = w.shape[1]
    if op == "conv_step":
        x = x[:, None]
    B, L, D = x.shape
    ends = [L] * B if lengths is None else lengths.tolist()
    alive = torch.tensor(ends, device=x.device)[:, None] > torch.arange(L, device=x.device)
    line = torch.cat([first, x.masked_fill(~alive[..., None], 0)], 1)
    pre = bias.expand(B, L, D).clone()
    for k in range(K):
        pre += line[:, k:k + L] * w[:, k]
    gate = 1 / (1 + (-pre).exp())
    y = (pre * gate).masked_fill(~alive[..., None], 0)
    last = torch.stack([line[r, e:e + K - 1] for r, e in enumerate(ends)])
    if op == "conv_step":
        return {"y": y[:, 0], "state": last}
    if op == "conv":
        return {"y": y, "state": last}
    dpre = (v["dy"] * (gate + pre * gate * (1 - gate))).masked_fill(~alive[..., None], 0)
    dline, dw = torch.zeros_like(line), torch.zeros_like(w)
    for k in range(K):
        dline[:, k:k + L] += dpre * w[:, k]
        dw[:, k] = (dpre * line[:, k:k + L]).sum((0, 1))
    return {"y": y, "last": last, "d_x": dline[:, K - 1:].masked_fill(~alive[..., None], 0), "d_weight": dw, "d_bias": dpre.sum((0, 1)),
            "d_state": dline[:, :K - 1]}


def _exact_scan(op, v, lengths):
    x, A, state = v["x"], v["A"], v["state"].clone()
    if op == "scan_step":
        x = x[:, None]
        v = {**v, **{k: v[k][:, None] for k in ("dt", "B", "C")}}
    rows, L, H, P = x.shape
    G, N = v["B"].shape[2:]
    train = op == "scan_train"
    if train and rows * L * H * P * N * 8 > 40e9:
        return None
    raw = v["dt"] + v["dt_bias"]
    dt = torch.where(raw > 30, raw, raw.exp().log1p())
    alive = torch.ones(rows, L, dtype=torch.bool, device=x.device)
    if lengths is not None:
        alive = lengths[:, None] > torch.arange(L, device=x.device)
    dt = dt * alive[..., None]
    head = torch.arange(H, device=x.device) // (H // G)
    y, kept = torch.empty_like(x), []
    factor = (dt * A).exp()[..., None, None]
    for t in range(L):
        kept.append(state) if train else None
        state = factor[:, t] * state + (dt[:, t, :, None] * x[:, t])[..., None] * v["B"][:, t, head][:, :, None]
        y[:, t] = (state @ v["C"][:, t, head][..., None])[..., 0]
    y = (y + v["D"][:, None] * x) * alive[..., None, None]
    if op == "scan_step":
        return {"y": y[:, 0], "state": state}
    if not train:
        return {"y": y, "state": state}
    dy = v["dy"] * alive[..., None, None]
    grad, now = v["dstate"].clone(), state
    d = {k: torch.zeros_like(v[k]) for k in ("x", "dt", "A", "B", "C")}
    for t in reversed(range(L)):
        b, c, step = v["B"][:, t, head], v["C"][:, t, head], dt[:, t]
        d["C"][:, t] = (dy[:, t, :, None] @ now)[:, :, 0].unflatten(1, (G, H // G)).sum(2)
        grad = grad + dy[:, t, :, :, None] * c[:, :, None]
        through = (grad @ b[..., None])[..., 0]
        d["B"][:, t] = (step[..., None] * (x[:, t, :, None] @ grad)[:, :, 0]).unflatten(1, (G, H // G)).sum(2)
        d["x"][:, t] = step[..., None] * through
        rate = (grad * kept[t]).sum((-1, -2)) * factor[:, t, :, 0, 0]
        d["dt"][:, t] = rate * A + (through * x[:, t]).sum(-1)
        d["A"] += (rate * step).sum(0)
        grad = grad * factor[:, t]
        now = kept[t]
    d["x"] += v["D"][:, None] * dy
    d["dt"] = d["dt"] * alive[..., None] / (1 + (-raw).exp())
    return {"y": y, "last": state, "d_x": d["x"], "d_dt": d["dt"], "d_A": d["A"], "d_B": d["B"], "d_C": d["C"],
            "d_D": (dy * x).sum((0, 1, 3)), "d_dt_bias": d["dt"].sum((0, 1)), "d_state": grad}
