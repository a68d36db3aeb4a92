"""rtfs_net_amd.ssm (csrc/ssm_conv.hip, ssm_scan.hip, ssm_bwd.hip) against token-by-token definitions in float64.

Tolerances (relative L2 error of a whole tensor), from the roundings counted: u = finfo.eps / 2 of the type.
  fp32: sums of at most 128 + 64 + a few products, each rounded once: below 256 u = 1.6e-5.
  bf16: y and dx: scores (or weights), state and result are rounded once each, 3 u; dB, dC: scores and result, 2 u; all inputs are exact.
  fp32 results of bf16 inputs (states, parameter gradients, dt's gradient): operands split to 2^-17, twice on the way: 256 u(fp32) + 2 * 2^-17 = 3.1e-5."""
import pytest
import torch

gpu = pytest.mark.gpu
U16, U32 = torch.finfo(torch.bfloat16).eps / 2, torch.finfo(torch.float32).eps / 2


def tol(kind, roundings=0):
    """`roundings` to bf16 when the inputs are; 0: a result that stays fp32"""
    if kind == torch.float32:
        return 256 * U32
    return roundings * U16 if roundings else 256 * U32 + 2 * 2.0 ** -17


def off(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    return float((got - want).norm() / want.norm().clamp_min(1e-30)) if want.numel() else 0.0


def alive_of(lengths, B, L):
    ends = torch.full((B,), L) if lengths is None else lengths.clamp(0, L).long()
    return ends, torch.arange(L) < ends[:, None]


def ref_conv(x, w, bias, state, lengths, silu):
    B, L, D = x.shape
    K = w.shape[1]
    ends, alive = alive_of(lengths, B, L)
    x = torch.where(alive[..., None], x, torch.zeros((), dtype=x.dtype))
    line = torch.cat([x.new_zeros(B, K - 1, D) if state is None else state, x], 1)
    pre = sum(line[:, k:k + L] * w[:, k] for k in range(K))
    if bias is not None:
        pre = pre + bias
    y = pre * torch.sigmoid(pre) if silu else pre
    return torch.where(alive[..., None], y, torch.zeros((), dtype=y.dtype)), torch.stack([line[b, e:e + K - 1] for b, e in enumerate(ends.tolist())])


def ref_scan(x, dt, A, Bm, C, D, bias, softplus, state, lengths):
    B, L, H, P = x.shape
    G, N = Bm.shape[2:]
    _, alive = alive_of(lengths, B, L)
    zero = torch.zeros((), dtype=x.dtype)
    x, Bm, C = (torch.where(alive[..., None, None], v, zero) for v in (x, Bm, C))
    d = torch.where(alive[..., None], dt, zero)
    d = d if bias is None else d + bias
    d = torch.nn.functional.softplus(d, threshold=60) if softplus else d
    d = torch.where(alive[..., None], d, zero)
    Bm, C = Bm.repeat_interleave(H // G, 2), C.repeat_interleave(H // G, 2)
    S = x.new_zeros(B, H, P, N) if state is None else state
    ys = []
    for t in range(L):
        S = torch.exp(d[:, t] * A)[..., None, None] * S + (d[:, t, :, None] * x[:, t])[..., None] * Bm[:, t, :, None]
        ys.append((S * C[:, t, :, None]).sum(-1))
    y = torch.stack(ys, 1)
    y = y if D is None else y + D[:, None] * x
    return torch.where(alive[..., None, None], y, zero), S


def scan_inputs(B, L, H, G, P, N, kind, seed=0, fp32_dt=False, pad=0):
    """on the CPU; `pad`: extra values per token, so that the tensors are slices"""
    r = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=kind):
        return (torch.randn(*shape, generator=r) * scale).to(dtype)

    v = {"x": normal(B, L, H * P + pad)[..., pad // 2:pad // 2 + H * P].unflatten(-1, (H, P)),
         "dt": normal(B, L, H + pad, scale=0.5, dtype=torch.float32 if fp32_dt else kind)[..., :H],
         "A": -(0.5 + 8 * torch.rand(H, generator=r)),
         "Bm": normal(B, L, G * N + pad)[..., :G * N].unflatten(-1, (G, N)), "C": normal(B, L, G * N + pad)[..., pad:].unflatten(-1, (G, N)),
         "D": 1 + normal(H, scale=0.1, dtype=torch.float32), "bias": normal(H, dtype=torch.float32) - 2,
         "state": normal(B, H, P, N, dtype=torch.float32)}
    return v


def gpu_scan(v, lengths=None, softplus=True, want_state=True):
    from rtfs_net_amd.ssm import selective_scan

    return selective_scan(v["x"], v["dt"], v["A"], v["Bm"], v["C"], v["D"], dt_bias=v["bias"], softplus=softplus, state=v["state"],
                          lengths=None if lengths is None else lengths.cuda(), return_state=want_state)


def cuda(v, leaf=False):
    """to the GPU with the same strides (slices stay slices)"""
    out = {}
    for k, t in v.items():
        if t is None:
            out[k] = None
            continue
        base = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
        out[k] = base.copy_(t).requires_grad_(leaf)
    return out


SHAPES = [  # B, L, H, G, P, N
    (1, 1, 1, 1, 1, 1), (2, 2, 4, 2, 32, 32), (3, 63, 2, 1, 17, 5), (2, 64, 4, 4, 64, 64), (1, 65, 2, 1, 128, 128), (2, 130, 6, 2, 48, 40),
    (5, 200, 3, 1, 33, 128), (1, 64 * 9 + 5, 2, 2, 64, 16), (2, 320, 4, 1, 20, 65), (1, 1030, 1, 1, 100, 33),
    (2, 130, 5, 1, 66, 9), (1, 200, 8, 1, 64, 128), (1, 128, 12, 3, 24, 64), (1, 70, 16, 1, 128, 100), (4, 190, 7, 7, 96, 31),
]


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_matches_the_recurrence(shape, kind):
    B, L, H, G, P, N = shape
    for pad, ragged in ((0, False), (24, True)):
        v = scan_inputs(*shape, kind, seed=L, pad=pad)
        lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(1), dtype=torch.int32) if ragged else None
        want, last = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, v["state"].double(), lengths)
        y, s = gpu_scan(cuda(v), lengths)
        assert y.dtype == kind and s.dtype == torch.float32
        assert off(y, want) <= tol(kind, 3) and off(s, last) <= tol(kind), (pad, off(y, want), off(s, last))
        assert torch.equal(gpu_scan(cuda(v), lengths, want_state=False), y)


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_gradients_match_the_recurrences(shape, kind):
    B, L, H, G, P, N = shape
    v = scan_inputs(*shape, kind, seed=L + 1, fp32_dt=L % 2 == 0)
    r = torch.Generator().manual_seed(2)
    lengths = torch.randint(0, L + 1, (B,), generator=r, dtype=torch.int32) if B > 2 else None
    dy, ds = torch.randn(B, L, H, P, generator=r).to(kind), torch.randn(B, H, P, N, generator=r)
    leaves = {k: t.double().requires_grad_() for k, t in v.items()}
    y, s = ref_scan(*(leaves[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, leaves["state"], lengths)
    want = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy.double(), ds.double()))))
    here = cuda(v, leaf=True)
    got = dict(zip(here, torch.autograd.grad(gpu_scan(here, lengths), list(here.values()), (dy.cuda(), ds.cuda()))))
    # One number has no random signs to average: dC = e^s S dy + (V E d) B with the second factor rounded is off by u |V E d B| + u |dC|, and |dC| may be as small
    # as the two terms happen to cancel.  Its error counts against the sum of the terms' magnitudes, which the same gradients of |inputs| give.
    size = want
    if B * L * H * P * N == 1:
        mag = {k: t.double().abs().requires_grad_() if k in ("x", "Bm", "C", "state", "D") else t.double().requires_grad_() for k, t in v.items()}
        m = ref_scan(*(mag[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, mag["state"], lengths)
        size = dict(zip(mag, torch.autograd.grad(m, list(mag.values()), (dy.double().abs(), ds.double().abs()))))
    bad = {}
    for k in want:
        assert got[k].dtype == v[k].dtype
        bound = {"x": tol(kind, 3), "Bm": tol(kind, 2), "C": tol(kind, 2), "dt": tol(kind, 0) if got[k].dtype == torch.float32 else tol(kind, 1) * 1.01}.get(k, tol(kind))
        # a sum over all tokens may cancel: its error counts against the sum of magnitudes, which for these inputs is below sqrt(tokens) of its value
        if k in ("A", "D", "bias"):
            bound *= max(1.0, (B * L * P) ** 0.5 / 8)
        err = off(got[k], want[k]) * float(want[k].norm() / size[k].norm())
        if err > bound:
            bad[k] = (err, bound)
    assert not bad, bad


@gpu
def test_scan_gradient_against_differences():
    """the loss moves along a random direction as the gradients say, by central differences of the float64 definition"""
    v = scan_inputs(2, 70, 4, 2, 24, 12, torch.float32, seed=5)
    r = torch.Generator().manual_seed(3)
    dy, way = torch.randn(2, 70, 4, 24, generator=r).double(), {k: torch.randn(t.shape, generator=r).double() * 0.3 for k, t in v.items()}
    here = cuda(v, leaf=True)
    grads = torch.autograd.grad(gpu_scan(here, want_state=False), list(here.values()), dy.float().cuda())
    got = sum(float((g.double().cpu() * way[k]).sum()) for k, g in zip(here, grads))

    def loss(h):
        w = {k: t.double() + h * way[k] for k, t in v.items()}
        return float((ref_scan(*(w[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, w["state"], None)[0] * dy).sum())

    want = (8 * (loss(1e-4) - loss(-1e-4)) - (loss(2e-4) - loss(-2e-4))) / 12e-4
    scale = sum(float((g.double().cpu() * way[k]).norm()) for k, g in zip(here, grads))
    assert abs(got - want) <= 256 * U32 * scale + 1e-7 * abs(want)


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,H,G,P,N,pad", [(1, 4, 1, 32, 32, 0), (3, 6, 2, 48, 40, 0), (2, 3, 3, 33, 7, 0), (2, 2, 1, 128, 128, 0), (1, 1, 1, 1, 1, 0), (2, 4, 2, 20, 12, 3),
                                           (3, 2, 1, 16, 100, 4)])
def test_prompt_in_pieces_then_single_tokens(kind, B, H, G, P, N, pad):
    """a prompt cut anywhere, then one token at a time, is the whole sequence; the conv goes on the same way"""
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

    L = 150
    v = scan_inputs(B, L, H, G, P, N, kind, seed=9, pad=pad)
    want, last = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, v["state"].double(), None)
    c = cuda(v)
    ys, state = [], c["state"]
    with torch.no_grad():
        for a, b in ((0, 64), (64, 65), (65, 147)):
            y, state = selective_scan(c["x"][:, a:b], c["dt"][:, a:b], c["A"], c["Bm"][:, a:b], c["C"][:, a:b], c["D"], dt_bias=c["bias"], softplus=True, state=state,
                                      return_state=True)
            ys.append(y)
        for t in range(147, L):
            ys.append(selective_scan_step(c["x"][:, t], c["dt"][:, t], c["A"], c["Bm"][:, t], c["C"][:, t], state, c["D"], dt_bias=c["bias"], softplus=True)[:, None])
    assert off(torch.cat(ys, 1), want) <= tol(kind, 3) and off(state, last) <= 2 * tol(kind)
    r = torch.Generator().manual_seed(4)
    D, K = H * P, 4
    x, w, b = torch.randn(B, 20, D, generator=r).to(kind), torch.randn(D, K, generator=r), torch.randn(D, generator=r)
    want, last = ref_conv(x.double(), w.double(), b.double(), None, None, True)
    xc, wc, bc = x.cuda(), w.cuda(), b.cuda()
    y0, s = causal_conv(xc[:, :2], wc, bc, return_state=True)
    y1, s = causal_conv(xc[:, 2:17], wc, bc, state=s, return_state=True)
    y2 = [causal_conv_step(xc[:, t], s, wc, bc)[:, None] for t in range(17, 20)]
    assert off(torch.cat([y0, y1, *y2], 1), want) <= tol(kind, 1) and torch.equal(s.cpu(), last.to(kind))


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,L,D,K,silu,pad", [(1, 1, 1, 1, True, 0), (2, 3, 5, 8, True, 0), (3, 70, 64, 4, True, 0), (2, 33, 40, 3, False, 8), (1, 300, 24, 4, True, 3),
                                              (4, 129, 512, 2, True, 0), (2, 2, 16, 5, True, 0), (7, 37, 192, 6, False, 0), (1, 40, 700, 7, True, 0), (2, 45, 64, 1, True, 0),
                                              (2, 45, 64, 8, True, 0), (1, 9, 8, 5, True, 0)])
def test_conv_and_its_gradients(kind, B, L, D, K, silu, pad):
    from rtfs_net_amd.ssm import causal_conv

    r = torch.Generator().manual_seed(L)
    for ragged, with_state in ((False, False), (True, True)):
        x = torch.randn(B, L, D + pad, generator=r).to(kind)[..., pad:]
        w, b = torch.randn(D, K, generator=r) / K ** 0.5, torch.randn(D, generator=r)
        state = torch.randn(B, K - 1, D, generator=r).to(kind) if with_state else None
        lengths = torch.randint(0, L + 1, (B,), generator=r, dtype=torch.int32) if ragged else None
        dy, dl = torch.randn(B, L, D, generator=r).to(kind), torch.randn(B, K - 1, D, generator=r).to(kind)
        leaves = {"x": x, "w": w, "b": b, **({"state": state} if with_state else {})}
        ref = {k: t.double().requires_grad_() for k, t in leaves.items()}
        y, last = ref_conv(ref["x"], ref["w"], ref["b"], ref.get("state"), lengths, silu)
        want = torch.autograd.grad((y, last), list(ref.values()), (dy.double(), dl.double()), allow_unused=True)
        here = cuda(leaves, leaf=True)
        out = causal_conv(here["x"], here["w"], here["b"], silu=silu, state=here.get("state"), lengths=None if lengths is None else lengths.cuda(), return_state=True)
        assert off(out[0], y) <= tol(kind, 1) and torch.equal(out[1].cpu().double(), last.detach())
        got = torch.autograd.grad(out, list(here.values()), (dy.cuda(), dl.cuda()))
        for k, g, q in zip(leaves, got, want):
            # w and b: fp32 sums over B L tokens whose magnitudes add up to at most sqrt(B L) of the result for random signs
            bound = tol(kind, 1) if k in ("x", "state") else 64 * U32 * max(1.0, (B * L) ** 0.5)
            assert off(g, torch.zeros_like(g, device="cpu") if q is None else q) <= bound, (k, ragged, off(g, q))


@gpu
def test_addresses_off_16_bytes():
    """every tensor a few values into its storage: the bits of aligned ones"""
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step, selective_scan_step

    def shifted(t):
        return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)

    for kind in (torch.float32, torch.bfloat16):
        x, w, b, s = torch.randn(2, 40, 64, device="cuda").to(kind), torch.randn(64, 4, device="cuda"), torch.randn(64, device="cuda"), torch.randn(2, 3, 64, device="cuda").to(kind)
        for off_x, off_w in ((True, False), (False, True), (True, True)):
            (p, u), (q, c, t) = (shifted(v) if off_x else v.clone() for v in (x, s)), (shifted(w) if off_w else w, shifted(b) if off_w else b, s.clone())
            for p0, p1 in zip(causal_conv(x, w, b, state=s, return_state=True), causal_conv(p, q, c, state=u, return_state=True)):
                assert torch.equal(p0, p1)
            assert torch.equal(causal_conv_step(x[:, 0], t, w, b), causal_conv_step(p[:, 0], u, q, c)) and torch.equal(t, u)
        v = cuda(scan_inputs(2, 100, 4, 2, 32, 32, kind, seed=15))
        m = {k: shifted(t) for k, t in v.items()}
        y, z = gpu_scan(v), gpu_scan(m)
        assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
        s0, s1 = v["state"].clone(), v["state"].clone()
        names = [(u["x"][:, 0], u["dt"][:, 0], u["A"], u["Bm"][:, 0], u["C"][:, 0]) for u in (v, m)]
        assert torch.equal(selective_scan_step(*names[0], s0), selective_scan_step(*names[1], s1)) and torch.equal(s0, s1)


@gpu
def test_nothing_behind_a_rows_end_is_read():
    """a padded batch may hold anything there: outputs, gradients and states are those of a batch of zeros there"""
    from rtfs_net_amd.ssm import causal_conv

    v = scan_inputs(4, 100, 2, 1, 16, 8, torch.float32, seed=1)
    lengths = torch.tensor([100, 37, 0, 64], dtype=torch.int32)
    _, alive = alive_of(lengths, 4, 100)
    results = []
    for filler in (0.0, float("nan"), float("inf")):
        w = {k: t.clone() for k, t in v.items()}
        for k in ("x", "dt", "Bm", "C"):
            w[k][~alive] = filler
        here = cuda(w, leaf=True)
        dy = torch.randn(4, 100, 2, 16, generator=torch.Generator().manual_seed(0))
        dy[~alive] = filler
        y, s = gpu_scan(here, lengths)
        results.append([y.detach(), s.detach(), *torch.autograd.grad((y, s), list(here.values()), (dy.cuda(), torch.ones_like(s)))])
        x = here["x"].detach().flatten(2).requires_grad_()
        wt = torch.randn(32, 4, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
        y, s = causal_conv(x, wt, lengths=lengths.cuda(), return_state=True)
        results[-1] += [y.detach(), s.detach(), *torch.autograd.grad((y, s), (x, wt), (dy.flatten(2).cuda(), torch.ones_like(s)))]
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    assert not results[0][0].cpu()[~alive].any()


@gpu
def test_rows_are_independent_and_runs_repeat():
    """a NaN in one row stays in it; the same inputs give the same bits, gradients included"""
    v = scan_inputs(3, 700, 2, 1, 32, 32, torch.bfloat16, seed=2)
    here = cuda(v, leaf=True)
    dy = torch.randn(3, 700, 2, 32, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()

    def once(v):
        y, s = gpu_scan(v)
        return [y.detach(), s.detach(), *torch.autograd.grad((y, s), list(v.values()), (dy, torch.ones_like(s)))]

    a, b = once(here), once(here)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    w = {k: t.clone() for k, t in v.items()}
    w["x"][1, 300, 0, 3] = float("nan")
    c = once(cuda(w, leaf=True))
    for p, q in zip(a[:2], c[:2]):
        assert torch.equal(p[0], q[0]) and torch.equal(p[2], q[2]) and q[1].isnan().any()


@gpu
def test_strong_decay_and_growth_stay_finite():
    """steps so large that every state is forgotten at once, and steps of zero: no NaN from differences of large sums, values by the definition"""
    v = scan_inputs(2, 200, 2, 1, 16, 16, torch.float32, seed=3)
    v["bias"] = torch.tensor([40.0, -300.0])
    want, last = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, v["state"].double(), None)
    y, s = gpu_scan(cuda(v))
    assert off(y, want) <= tol(torch.float32) and off(s, last) <= tol(torch.float32)
    v = scan_inputs(1, 130, 2, 1, 16, 16, torch.float32, seed=4)
    v["A"], v["bias"] = torch.tensor([0.05, 0.0]), torch.zeros(2)  # a state that grows, one that only adds up
    want, last = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, v["state"].double(), None)
    y, s = gpu_scan(cuda(v))
    assert off(y, want) <= 4 * tol(torch.float32) and off(s, last) <= 4 * tol(torch.float32)


@gpu
def test_optional_arguments():
    """without D, bias, softplus, state; one output alone wanted, one gradient alone given"""
    from rtfs_net_amd.ssm import selective_scan

    v = scan_inputs(2, 90, 2, 1, 16, 16, torch.float32, seed=6)
    v["dt"] = v["dt"].abs() * 0.1
    leaves = {k: v[k].double().requires_grad_() for k in ("x", "dt", "A", "Bm", "C")}
    y, s = ref_scan(*leaves.values(), None, None, False, None, None)
    here = cuda({k: v[k] for k in leaves}, leaf=True)
    for pick in (0, 1):
        want = torch.autograd.grad((y, s)[pick].square().sum(), list(leaves.values()), retain_graph=True, allow_unused=True)
        out = selective_scan(*here.values(), return_state=True)[pick]
        got = torch.autograd.grad(out.square().sum(), list(here.values()))
        for k, a, b in zip(leaves, got, want):
            assert off(a, torch.zeros(a.shape) if b is None else b) <= 8 * tol(torch.float32), (pick, k)
    assert torch.equal(selective_scan(*(t.detach() for t in here.values())), selective_scan(*here.values()).detach())


@gpu
def test_no_state_is_a_state_of_zeros():
    """nothing of what a call does not ask for is needed by the rest of it, in rows of one segment and of many"""
    for B, L in ((1, 64), (1, 1030), (300, 130)):
        v = scan_inputs(B, L, 4, 2, 32, 24, torch.bfloat16, seed=14)
        v["state"].zero_()
        here = cuda(v, leaf=True)
        names = [k for k in here if k != "state"]
        y, s = gpu_scan(here)
        want = torch.autograd.grad(y, [here[k] for k in names], torch.ones_like(y))
        z = gpu_scan({**here, "state": None}, want_state=False)
        got = torch.autograd.grad(z, [here[k] for k in names], torch.ones_like(z))
        assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(want, got)), (B, L)


@gpu
@pytest.mark.parametrize("B,L", [(0, 5), (2, 0)])
def test_no_tokens(B, L):
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step, selective_scan_step

    v = cuda(scan_inputs(B, L, 2, 1, 4, 4, torch.float32))
    y, s = gpu_scan(v)
    assert y.shape == (B, L, 2, 4) and torch.equal(s, v["state"])
    w = torch.ones(8, 4, device="cuda")
    y, s = causal_conv(v["x"].flatten(2), w, return_state=True)
    assert y.shape == (B, L, 8) and s.shape == (B, 3, 8) and not s.any()
    if B == 0:
        assert causal_conv_step(v["x"].new_zeros(0, 8), w.new_zeros(0, 3, 8), w).shape == (0, 8)
        assert selective_scan_step(w.new_zeros(0, 2, 4), w.new_zeros(0, 2), v["A"], w.new_zeros(0, 1, 4), w.new_zeros(0, 1, 4), v["state"]).shape == (0, 2, 4)


@gpu
def test_captured_steps_and_prompts_replay():
    """two graphs captured from the same calls, replayed in turn with eager work between, give the eager results each time"""
    from rtfs_net_amd.ssm import causal_conv_step, selective_scan_step

    r = torch.Generator(device="cuda").manual_seed(0)
    x, dt = torch.empty(2, 1, 4, 16, device="cuda"), torch.empty(2, 1, 4, device="cuda")
    A, w = -torch.rand(4, device="cuda", generator=r), torch.randn(64, 4, device="cuda", generator=r)
    bc = torch.randn(2, 1, 1, 8, device="cuda", generator=r)
    long = cuda(scan_inputs(1, 64 * 12, 2, 1, 32, 32, torch.float32, seed=8))

    def token(conv, state):
        y = causal_conv_step(x.view(2, 64), conv, w)
        return selective_scan_step(y.view(2, 4, 16), dt[:, 0], A, bc[:, 0], bc[:, 0], state, softplus=True)

    def fresh():
        return torch.zeros(2, 3, 64, device="cuda"), torch.zeros(2, 4, 16, 8, device="cuda")

    eager, held = fresh(), fresh()
    x.normal_(generator=r), dt.normal_(generator=r)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), torch.no_grad():
        token(*fresh()), gpu_scan(long)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(one):
            out = token(*held)
        with torch.cuda.graph(two):
            prompt = gpu_scan(long)
    held[0].zero_(), held[1].zero_()
    for i in range(4):
        x.normal_(generator=r), dt.normal_(generator=r)
        long["x"].normal_(generator=r)
        one.replay()
        want = token(*eager)
        two.replay()
        y, s = gpu_scan(long)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1]), i
        assert torch.equal(prompt[0], y) and torch.equal(prompt[1], s), i


@gpu
def test_a_layer_of_them_trains_and_serves():
    """projection -> convolution -> scan, a training step with the clip, on a side stream; then the trained layer frame by frame gives the prompt's outputs"""
    from rtfs_net_amd.optim import clip_grad_norm_
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

    torch.manual_seed(0)
    H, P, N, dim = 4, 32, 16, 64
    width = H * P + 2 * N
    into, weight, A = torch.nn.Linear(dim, width + H).cuda(), torch.nn.Parameter(torch.randn(width, 4, device="cuda") / 2), torch.nn.Parameter(torch.zeros(H, device="cuda"))
    params = [*into.parameters(), weight, A]
    opt = torch.optim.SGD(params, lr=0.1)

    def layer(x):
        xbc, dt = into(x).split([width, H], -1)
        xs, b, c = causal_conv(xbc, weight).split([H * P, N, N], -1)
        return selective_scan(xs.unflatten(-1, (H, P)), dt, -A.exp(), b[:, :, None], c[:, :, None], softplus=True)

    x = torch.randn(3, 150, dim, device="cuda")
    before = [p.detach().clone() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x).square().mean().backward()
        grads = [p.grad.clone() for p in params]
        norm = clip_grad_norm_(params, 1e-3)
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    want = torch.stack([g.double().norm() for g in grads]).norm()
    assert abs(float(norm) / float(want) - 1) < 4 * U32 and float(want) > 1e-3
    for p, q, g in zip(params, before, grads):
        assert g.abs().max() > 0 and off(p.grad, g * (1e-3 / (norm + 1e-6))) <= 4 * U32
        assert torch.equal(p.detach(), torch.add(q, p.grad, alpha=-0.1))
    with torch.no_grad():
        want = layer(x)
        xbc, dt = into(x).split([width, H], -1)
        conv, state, got = torch.zeros(3, 3, width, device="cuda"), torch.zeros(3, H, P, N, device="cuda"), []
        for t in range(150):
            xs, b, c = causal_conv_step(xbc[:, t], conv, weight).split([H * P, N, N], -1)
            got.append(selective_scan_step(xs.unflatten(-1, (H, P)), dt[:, t], -A.exp(), b[:, None], c[:, None], state, softplus=True))
    assert off(torch.stack(got, 1), want) <= 2 * tol(torch.float32)


@gpu
def test_broadcast_inputs_get_summed_gradients():
    """B and C expanded over the rows (stride 0) are read in place and their gradients summed"""
    v = scan_inputs(3, 70, 2, 1, 16, 16, torch.float32, seed=7)
    one = {**v, "Bm": v["Bm"][:1], "C": v["C"][:1]}
    leaves = {k: t.double().requires_grad_() for k, t in one.items()}
    full = {**leaves, "Bm": leaves["Bm"].expand(3, -1, -1, -1), "C": leaves["C"].expand(3, -1, -1, -1)}
    y, _ = ref_scan(*(full[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, full["state"], None)
    want = torch.autograd.grad(y.sum(), [leaves["Bm"], leaves["C"]])
    here = cuda(one, leaf=True)
    out, _ = gpu_scan({**here, "Bm": here["Bm"].expand(3, -1, -1, -1), "C": here["C"].expand(3, -1, -1, -1)})
    got = torch.autograd.grad(out.sum(), [here["Bm"], here["C"]])
    assert all(off(a, b) <= tol(torch.float32) for a, b in zip(got, want))


@gpu
def test_lengths_outside_the_batch_are_clamped():
    from rtfs_net_amd.ssm import causal_conv

    v = cuda(scan_inputs(3, 80, 2, 1, 16, 8, torch.float32, seed=11))
    far, near = torch.tensor([-5, 300, 2 ** 31 - 1], dtype=torch.int32), torch.tensor([0, 80, 80], dtype=torch.int32)
    assert all(torch.equal(a, b) for a, b in zip(gpu_scan(v, far), gpu_scan(v, near)))
    x, w = v["x"].flatten(2), torch.randn(32, 4, device="cuda")
    for a, b in zip(causal_conv(x, w, lengths=far.cuda(), return_state=True), causal_conv(x, w, lengths=near.cuda(), return_state=True)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("tok,L", [(1 << 22, 1100), (1 << 23, 70)])
def test_tokens_far_apart(tok, L):
    """slices of a wide bf16 tensor whose offsets pass 2^32 elements (and tokens too far apart for the kernels, which are copied together): the bits of dense inputs"""
    from rtfs_net_amd.ssm import causal_conv, selective_scan

    wide = torch.empty(1, L, tok, dtype=torch.bfloat16, device="cuda")
    wide[..., :132].normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    A, w = torch.tensor([-1.0, -4.0], device="cuda"), torch.randn(64, 4, device="cuda")

    def run(u):
        u = u.requires_grad_()
        y = selective_scan(u[..., :64].unflatten(-1, (2, 32)), u[..., 128:130], A, u[..., 64:96].unflatten(-1, (1, 32)), u[..., 96:128].unflatten(-1, (1, 32)),
                           softplus=True)
        z = causal_conv(u[..., :64], w)
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), u, (torch.ones_like(y), torch.ones_like(z)))]

    dense = run(wide[..., :132].contiguous())
    here = run(wide.detach()[..., :132])
    assert all(torch.equal(a, b) for a, b in zip(dense, here))


@gpu
def test_more_than_2_31_elements():
    """the last tokens of sequences whose tensors pass 2^31 elements are those of a call that starts in front of them"""
    from rtfs_net_amd.ssm import causal_conv, selective_scan

    r, kind = torch.Generator(device="cuda").manual_seed(0), torch.bfloat16
    L, H, P, N = 70016, 512, 64, 16
    cut = L - 64 * 20
    x = torch.randn(1, L, H, P, dtype=kind, device="cuda", generator=r)
    dt = torch.randn(1, L, H, device="cuda", generator=r) * 0.5 - 2
    bc = torch.randn(2, 1, L, 1, N, dtype=kind, device="cuda", generator=r)
    A = -1 - torch.rand(H, device="cuda", generator=r)
    dy = torch.zeros(1, L, H, P, dtype=kind, device="cuda")
    dy[:, cut:].normal_(generator=r)
    with torch.no_grad():
        _, state = selective_scan(x[:, :cut], dt[:, :cut], A, bc[0, :, :cut], bc[1, :, :cut], softplus=True, return_state=True)

    def run(a, state):
        leaves = [t.detach().requires_grad_() for t in (x[:, a:], dt[:, a:], bc[0, :, a:], bc[1, :, a:])]
        y, s = selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3], softplus=True, state=state, return_state=True)
        grads = torch.autograd.grad(y, leaves, dy[:, a:])
        return [t[:, cut - a:].clone() for t in (y.detach(), *grads)] + [s]

    for a, b, bound in zip(run(0, None), run(cut, state), (6 * U16, 6 * U16, tol(kind), 4 * U16, 4 * U16, tol(kind))):
        assert off(a, b) <= 2 * bound
    x = torch.randn(1, (1 << 21) + 70, 1024, dtype=kind, device="cuda", generator=r)
    w = torch.randn(1024, 4, device="cuda", generator=r)
    dy = torch.zeros_like(x)
    dy[:, -200:].normal_(generator=r)
    u, t = x.requires_grad_(), x.detach()[:, -200:].requires_grad_()
    y, z = causal_conv(u, w), causal_conv(t, w, state=x.detach()[:, -203:-200])
    du, dz = torch.autograd.grad(y, u, dy)[0], torch.autograd.grad(z, t, dy[:, -200:])[0]
    assert torch.equal(y[:, -200:], z) and torch.equal(du[:, -200:], dz)


@gpu
@pytest.mark.parametrize("K", range(1, 9))
def test_single_tokens_of_every_width(K):
    """prompt and single tokens give the same bits, and the same state, for each number of taps"""
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step

    for kind, D in ((torch.float32, 64), (torch.bfloat16, 64), (torch.float32, 33), (torch.bfloat16, 33)):
        x, w = torch.randn(3, 12, D, device="cuda").to(kind), torch.randn(D, K, device="cuda")
        want, last = causal_conv(x, w, return_state=True)
        state = torch.zeros(3, K - 1, D, dtype=kind, device="cuda")
        got = torch.stack([causal_conv_step(x[:, t], state, w) for t in range(12)], 1)
        assert torch.equal(got, want) and torch.equal(state, last)


@gpu
def test_many_rows():
    from rtfs_net_amd.ssm import causal_conv_step, selective_scan, selective_scan_step

    B, P = (1 << 22) - 1, 100
    x = torch.randn(B, 1, 1, P, device="cuda")
    dt, A, bc, s = torch.rand(B, 1, 1, device="cuda"), torch.tensor([-1.0], device="cuda"), torch.randn(2, B, 1, 1, 1, device="cuda"), torch.ones(B, 1, P, 1, device="cuda")
    y, last = selective_scan(x, dt, A, bc[0], bc[1], state=s, return_state=True)
    one = selective_scan_step(x[:, 0], dt[:, 0], A, bc[0, :, 0], bc[1, :, 0], s)
    d = dt[:, :, :, None].double()
    want = torch.exp(-d) + d * x.double() * bc[0].double()
    for got in (last, s):
        assert float((got.view(B, 1, 1, P).double() - want).norm() / want.norm()) <= tol(torch.float32)
    want *= bc[1].double()
    for got in (y, one[:, None]):
        assert float((got.double() - want).norm() / want.norm()) <= tol(torch.float32)
    x = x.view(B, P)
    state, w = torch.ones(B, 1, P, device="cuda"), torch.ones(P, 2, device="cuda")
    assert torch.equal(causal_conv_step(x, state, w, silu=False), 1 + x) and torch.equal(state[:, 0], x)


@gpu
def test_serving_in_inference_mode():
    from rtfs_net_amd.ssm import causal_conv_step, selective_scan, selective_scan_step

    v = cuda(scan_inputs(2, 3, 2, 1, 16, 8, torch.bfloat16, seed=12))
    with torch.inference_mode():
        y, s = selective_scan(v["x"], v["dt"], v["A"], v["Bm"], v["C"], return_state=True)
        held = torch.zeros(2, 2, 16, 8, device="cuda")
        steps = [selective_scan_step(v["x"][:, t], v["dt"][:, t], v["A"], v["Bm"][:, t], v["C"][:, t], held) for t in range(3)]
        conv = torch.zeros(2, 3, 32, dtype=torch.bfloat16, device="cuda")
        causal_conv_step(v["x"][:, 0].flatten(1), conv, torch.ones(32, 4, device="cuda"))
    assert off(torch.stack(steps, 1), y) <= 2 * tol(torch.bfloat16, 3) and off(held, s) <= 2 * tol(torch.bfloat16)
    assert torch.equal(conv[:, 2], v["x"][:, 0].flatten(1))


@gpu
def test_calls_on_two_streams_at_once():
    """each call's workspaces are its own: interleaved on two streams they give the bits of one after the other"""
    v = [cuda(scan_inputs(1, 64 * 40, 2, 1, 64, 64, torch.float32, seed=s), leaf=True) for s in (0, 1)]
    dy = torch.randn(1, 64 * 40, 2, 64, device="cuda")

    def once(u):
        y, s = gpu_scan(u)
        return [y.detach(), s.detach(), *torch.autograd.grad((y, s), list(u.values()), (dy, torch.ones_like(s)))]

    want = [once(u) for u in v]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for u, st in zip(v, streams):
            with torch.cuda.stream(st):
                got.append(once(u))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


@gpu
def test_captured_training_step_replays():
    """convolution, scan and their gradients in one graph: each replay has the eager bits"""
    from rtfs_net_amd.ssm import causal_conv

    v = cuda(scan_inputs(2, 64 * 5 + 3, 4, 2, 32, 16, torch.bfloat16, seed=13), leaf=True)
    w = torch.randn(128, 4, device="cuda", requires_grad=True)
    dy = torch.randn(2, 64 * 5 + 3, 4, 32, device="cuda").bfloat16()
    leaves = [*v.values(), w]

    def step():
        x = causal_conv(v["x"].flatten(2), w).unflatten(-1, (4, 32))
        y, s = gpu_scan({**v, "x": x})
        return [y.detach(), s.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            for t in (v["x"], v["Bm"], v["C"], dy, w):
                t.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_refusals_of_the_convolution():
    from rtfs_net_amd.ssm import causal_conv, causal_conv_step

    x, w, s = torch.zeros(2, 5, 6), torch.zeros(6, 4), torch.zeros(2, 3, 6)
    for bad in (lambda: causal_conv(x[0], w), lambda: causal_conv(x.half(), w), lambda: causal_conv(x, torch.zeros(6, 9)), lambda: causal_conv(x, w[:5]),
                lambda: causal_conv(x, w.double()), lambda: causal_conv(x, w, torch.zeros(5)), lambda: causal_conv(x, w, state=s[:, :2]),
                lambda: causal_conv(x, w, state=s.bfloat16()), lambda: causal_conv(x, w, lengths=torch.zeros(2)),
                lambda: causal_conv(x, w, lengths=torch.zeros(3, dtype=torch.int32)), lambda: causal_conv_step(x[:, 0], s[:1], w),
                lambda: causal_conv_step(x[:, 0], s.transpose(1, 2).contiguous().transpose(1, 2), w), lambda: causal_conv_step(x, s, w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        causal_conv([1.0], w)
    with pytest.raises(RuntimeError, match="no gradient"):
        causal_conv_step(x[:, 0], s, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="HIP"):
        causal_conv(x, w)
    with pytest.raises(RuntimeError, match="HIP"):
        causal_conv_step(x[:, 0], s, w)


def test_refusals_of_the_scan():
    from rtfs_net_amd.ssm import selective_scan, selective_scan_step

    x, dt, A, bc, s = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 4), torch.zeros(4), torch.zeros(2, 5, 2, 3), torch.zeros(2, 4, 8, 3)
    wide = torch.zeros(2, 5, 2, 129)
    for bad in (lambda: selective_scan(x[0], dt, A, bc, bc), lambda: selective_scan(x.half(), dt, A, bc, bc), lambda: selective_scan(x, dt[:, :4], A, bc, bc),
                lambda: selective_scan(x, dt.bfloat16(), A, bc, bc), lambda: selective_scan(x, dt, A[:3], bc, bc), lambda: selective_scan(x, dt, A.double(), bc, bc),
                lambda: selective_scan(x, dt, A, bc, bc[..., :2]), lambda: selective_scan(x, dt, A, bc[:, :, :0], bc[:, :, :0]), lambda: selective_scan(x, dt, A, wide, wide),
                lambda: selective_scan(x[:, :, :3], dt[..., :3], A[:3], bc, bc), lambda: selective_scan(torch.zeros(2, 5, 4, 129), dt, A, bc, bc),
                lambda: selective_scan(x, dt, A, bc, bc, A[:2]), lambda: selective_scan(x, dt, A, bc, bc, dt_bias=A.bfloat16()),
                lambda: selective_scan(x, dt, A, bc, bc, state=s[:1]), lambda: selective_scan(x, dt, A, bc, bc, state=s.bfloat16()),
                lambda: selective_scan(x, dt, A, bc, bc, lengths=torch.zeros(2, dtype=torch.int64)), lambda: selective_scan(x, dt, A, bc.bfloat16(), bc),
                lambda: selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], None), lambda: selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], s.bfloat16()),
                lambda: selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], torch.zeros(2, 4, 3, 8).transpose(2, 3)),
                lambda: selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], torch.zeros(193)[1:].view(2, 4, 8, 3)),
                lambda: selective_scan(torch.zeros(1 << 20, 1, 4, 1), torch.zeros(1 << 20, 1, 4), A, torch.zeros(1 << 20, 1, 1, 1), torch.zeros(1 << 20, 1, 1, 1)),
                lambda: selective_scan(torch.zeros(1, 1, 1 << 17, 64), torch.zeros(1, 1, 1 << 17), torch.zeros(1 << 17), bc[:1, :1], bc[:1, :1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        selective_scan(x, None, A, bc, bc)
    with pytest.raises(RuntimeError, match="no gradient"):
        selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], s.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="HIP"):
        selective_scan(x, dt, A, bc, bc)
    with pytest.raises(RuntimeError, match="HIP"):
        selective_scan_step(x[:, 0], dt[:, 0], A, bc[:, 0], bc[:, 0], s)


def test_the_library_refuses_what_its_kernels_cannot_take():
    """sizes and types outside the contract come back as an error before anything is launched (no device is touched)"""
    from rtfs_net_amd import lib

    h = lib.load()
    one = 16  # an address that is never followed: the sizes are refused first
    scan = lambda *dims: h.rtfs_ssm_scan_fwd(one, 1, 1, one, 1, 1, 0, one, one, 1, 1, one, 1, 1, None, None, 0, None, None, one, None, None, *dims, None)  # noqa: E731
    for dims in ((0, 1, 1, 1, 1, 1, 0), (1, 0, 1, 1, 1, 1, 0), (1, 1, 3, 1, 2, 1, 0), (1, 1, 1, 129, 1, 1, 0), (1, 1, 1, 1, 1, 129, 0), (1, 1, 1, 1, 1, 1, 2)):
        assert scan(*dims) == -1
    assert scan(1, 4096, 1, 1, 1, 1, 0) == -1  # cut into segments, and no workspace for them
    conv = lambda *dims: h.rtfs_causal_conv_fwd(one, 1, 1, one, None, None, None, one, None, *dims, None)  # noqa: E731
    for dims in ((0, 1, 1, 1, 1, 0), (1, 1, 1, 9, 1, 0), (1, 1, 1, 0, 1, 0), (1, 1, 1, 1, 1, 3)):
        assert conv(*dims) == -1
    assert h.rtfs_ssm_tile(129, 1) == -1 and h.rtfs_ssm_tile(33, 65) == 64 * 128 and h.rtfs_causal_conv_bwd_work_floats(0, 4, 0) == -1
    assert h.rtfs_ssm_scan_segments(1, 64 * 100, 1, 16, 1, 16, 1) == 100 and h.rtfs_ssm_scan_segments(512, 64 * 100, 1, 16, 1, 16, 1) == 1 and h.rtfs_ssm_scan_bwd_parts(1, 64, 8, 3, 1) == -1


# A result that is off by d before it is rounded differs from the definition's rounded value only where a border lies between them: with probability |d| / step, by a
# step (2 U16 of the value at most), so its square adds up to sum |d| step <= |d| |step|.
BORDERS = (2 * U16 * tol(torch.bfloat16)) ** 0.5


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_bf16_outputs_are_the_definition_rounded_once(shape):
    """nothing inside a prompt is rounded to bf16 alone: y is the definition's rounded value but next to the borders between two"""
    v = scan_inputs(*shape, torch.bfloat16, seed=shape[1] + 1, fp32_dt=shape[1] % 2 == 0)
    want, _ = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, v["state"].double(), None)
    y, _ = gpu_scan(cuda(v))
    assert off(y, want.bfloat16()) <= BORDERS


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_bf16_gradients_are_the_definition_rounded_once(shape):
    B, L, H, G, P, N = shape
    v = scan_inputs(*shape, torch.bfloat16, seed=L + 1)
    r = torch.Generator().manual_seed(2)
    dy, ds = torch.randn(B, L, H, P, generator=r).bfloat16(), torch.randn(B, H, P, N, generator=r)
    leaves = {k: t.double().requires_grad_() for k, t in v.items()}
    y, s = ref_scan(*(leaves[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, leaves["state"], None)
    want = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy.double(), ds.double()))))
    here = cuda(v, leaf=True)
    got = dict(zip(here, torch.autograd.grad(gpu_scan(here), list(here.values()), (dy.cuda(), ds.cuda()))))
    far = {k: off(got[k], want[k].bfloat16()) for k in ("x", "dt", "Bm", "C")}
    assert max(far.values()) <= BORDERS, far


def test_one_token_has_no_pitch():
    """torch calls a time-first token contiguous and keeps the stride of the whole batch for it"""
    from rtfs_net_amd.ssm import _tokens

    x = torch.empty(1, 2048, 4, 1024).transpose(0, 1)
    assert x.is_contiguous() and x.stride(1) == 1 << 23
    t, row, tok = _tokens(x, 2)
    assert t is x and (row, tok) == (4096, 4096)


@gpu
def test_one_token_of_a_time_first_batch():
    from rtfs_net_amd.ssm import causal_conv, selective_scan

    r = torch.Generator(device="cuda").manual_seed(0)
    x, dt, bc = (torch.randn(1, 2048, *s, device="cuda", generator=r).transpose(0, 1) for s in ((32, 128), (32,), (1, 8)))
    A, w = -torch.rand(32, device="cuda", generator=r), torch.randn(4096, 2, device="cuda", generator=r)
    assert x.stride(1) >= 1 << 23

    def run(*leaves):
        leaves = [t.detach().requires_grad_() for t in leaves]
        y = selective_scan(*leaves[:2], A, leaves[2], leaves[2], softplus=True)
        z = causal_conv(leaves[0].flatten(2), w)
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), leaves, (torch.ones_like(y), torch.ones_like(z)))]

    dense = [torch.empty(t.shape, device="cuda").copy_(t) for t in (x, dt, bc)]
    assert dense[0].stride(1) < 1 << 23
    assert all(torch.equal(a, b) for a, b in zip(run(x, dt, bc), run(*dense)))


@gpu
@pytest.mark.parametrize("B,L", [(0, 5), (2, 0), (0, 0)])
def test_gradients_without_tokens(B, L):
    """an empty micro-batch trains on: zeros for the parameters, the last state's gradient for the given state"""
    from rtfs_net_amd.ssm import causal_conv, selective_scan

    v = cuda(scan_inputs(B, L, 2, 1, 4, 4, torch.float32), leaf=True)
    names = ("A", "Bm", "C", "D", "bias", "x", "dt")
    y, s = gpu_scan(v)
    ds = torch.randn_like(s)
    got = torch.autograd.grad((y, s), [v["state"], *(v[k] for k in names)], (torch.ones_like(y), ds))
    assert torch.equal(got[0], ds) and all(g.shape == v[k].shape and not g.any() for k, g in zip(names, got[1:]))
    x, A = v["x"].detach(), torch.zeros(2, device="cuda", requires_grad=True)
    selective_scan(x, v["dt"].detach(), A, v["Bm"].detach(), v["C"].detach()).sum().backward()
    assert not A.grad.any()
    w, b, c = (torch.randn(*n, device="cuda", requires_grad=True) for n in ((8, 4), (8,), (B, 3, 8)))
    y, s = causal_conv(x.flatten(2), w, b, state=c, return_state=True)
    ds = torch.randn_like(s)
    dw, db, dc = torch.autograd.grad((y, s), (w, b, c), (torch.ones_like(y), ds))
    assert not dw.any() and not db.any() and torch.equal(dc, ds)
    causal_conv(x.flatten(2), w).sum().backward()
    assert not w.grad.any() and w.grad.shape == w.shape
    none, empty = torch.zeros(2, 3, 0, device="cuda"), torch.zeros(0, 4, device="cuda", requires_grad=True)
    causal_conv(none, empty).sum().backward()
    assert empty.grad.shape == (0, 4)


def swings(up, down):
    """steps of both signs: six tokens that let states grow by e^up, twelve that let them fall by e^down, within one tile of 16 tokens and across three"""
    v = scan_inputs(2, 150, 2, 1, 16, 16, torch.float32, seed=3)
    v["A"], v["bias"] = torch.tensor([-1.0, -0.5]), torch.zeros(2)
    dt = torch.full((2, 150, 2), 0.05)
    for at in (8, 34, 118):
        dt[:, at:at + 6], dt[:, at + 6:at + 18] = -up / 6, down / 12
    v["dt"] = dt / -v["A"]
    return v


def per_token(got, want):
    got, want = got.detach().double().cpu(), want.detach().double()
    return (got - want).norm(dim=(2, 3)) / want.norm(dim=(2, 3))


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("up,down", [(60, 200), (80, 80), (75, 90)])
def test_steps_of_both_signs(kind, up, down):
    """states that fall and grow within a chunk: every token by the definition, and the gradients.  Exponents of up to 300 (log2) are rounded to fp32: 4 tol."""
    v = swings(up, down)
    v = {k: t.to(kind) if k in ("x", "Bm", "C") else t for k, t in v.items()}
    leaves = {k: t.double().requires_grad_() for k, t in v.items()}
    want = ref_scan(*(leaves[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), False, leaves["state"], None)
    here = cuda(v, leaf=True)
    got = gpu_scan(here, softplus=False)
    assert float(per_token(got[0], want[0]).max()) <= max(4 * tol(torch.float32), tol(kind, 1)) and off(got[1], want[1]) <= 4 * tol(kind)
    dy = torch.randn(want[0].shape, generator=torch.Generator().manual_seed(2)).to(kind)
    a = torch.autograd.grad(got[0], list(here.values()), dy.cuda())
    b = torch.autograd.grad(want[0], list(leaves.values()), dy.double())
    far = {}
    for k, p, q in zip(v, a, b):  # (a rate's gradient is 1.04e39 at 80 up and 80 down, more than fp32's largest 3.4e38: its rounding is an infinity of its sign)
        beyond = q.float().isinf()
        assert torch.equal(p.cpu().float()[beyond], q.float()[beyond]) and (k == "A" or not beyond.any())
        far[k] = off(p.cpu()[~beyond], q[~beyond])
    assert max(far.values()) <= max(8 * tol(torch.float32), tol(kind, 1)), far


@gpu
def test_states_beyond_fp32_for_a_while():
    """between tokens that are less than e^88 apart the outputs are right, also where the state passes fp32's range between them"""
    v = swings(120, 144)
    want, last = ref_scan(*(v[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), False, v["state"].double(), None)
    y, s = gpu_scan(cuda(v), softplus=False)
    far = per_token(y, want)
    ok = want.abs().amax((2, 3)) < 1e34
    assert ok[:, 60:118].all() and ok.float().mean() > 0.8
    assert float(far[ok].max()) <= 4 * tol(torch.float32) and off(s, last) <= 4 * tol(torch.float32)


@gpu
@pytest.mark.parametrize("rates", [(-1e38, -3e37), (-1e14, -1e9), (-3e38, -1.0)], ids=str)
def test_rates_that_forget_at_once(rates):
    """decays whose logarithms pass fp32's range, or leave no bits for the weaker ones behind them: prompt, gradients and single tokens by the definition"""
    from rtfs_net_amd.ssm import selective_scan_step

    v = scan_inputs(2, 70, 2, 1, 16, 16, torch.float32, seed=3)
    v["A"] = torch.tensor(rates)
    v["dt"][:, 1::2], v["bias"] = -200.0, torch.zeros(2)  # every other step is e^-200: 0 in fp32
    v["dt"][:, 5::6] = v["dt"][:, 4::6][:, :v["dt"][:, 5::6].shape[1]] - 20  # and some are e^-20 of their neighbour's
    leaves = {k: t.double().requires_grad_() for k, t in v.items()}
    want = ref_scan(*(leaves[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, leaves["state"], None)
    here = cuda(v, leaf=True)
    got = gpu_scan(here)
    assert off(got[0], want[0]) <= tol(torch.float32) and off(got[1], want[1]) <= tol(torch.float32)
    dy = torch.randn(want[0].shape, generator=torch.Generator().manual_seed(2))
    names = ("x", "Bm", "C", "D")
    for k, p, q in zip(names, torch.autograd.grad(got[0], [here[k] for k in names], dy.cuda()), torch.autograd.grad(want[0], [leaves[k] for k in names], dy.double())):
        assert off(p, q) <= tol(torch.float32), k
    u = {k: t.detach() for k, t in here.items()}
    state = u["state"].clone()
    steps = [selective_scan_step(u["x"][:, t], u["dt"][:, t], u["A"], u["Bm"][:, t], u["C"][:, t], state, u["D"], dt_bias=u["bias"], softplus=True) for t in range(70)]
    assert off(torch.stack(steps, 1), want[0]) <= tol(torch.float32) and off(state, want[1]) <= tol(torch.float32)


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 130, 4, 2, 32, 32), (2, 200, 2, 1, 100, 33), (600, 130, 2, 1, 17, 5), (2, 70, 3, 1, 64, 128), (2, 140, 2, 1, 64, 64), (5, 90, 1, 1, 128, 128)], ids=str)
def test_values_that_are_not_finite_go_forward_only(shape, kind):
    """an infinity or a NaN changes what the definition says depends on it, from its token on; everything else keeps its bits, the rest of its chunk included"""
    v = scan_inputs(*shape, kind, seed=7)
    y0, s0 = (t.cpu() for t in gpu_scan(cuda(v)))
    b, h = shape[0] - 1, shape[2] - 1
    for name, t, bad in (("x", 0, "nan"), ("x", 37, "nan"), ("x", 64, "inf"), ("x", 69, "-inf"), ("Bm", 50, "nan"), ("Bm", 65, "inf"), ("C", 33, "nan"), ("C", 64, "-inf"), ("dt", 47, "nan"),
                         ("dt", 66, "inf"), ("dt", 20, "-inf"), ("state", 0, "nan")):
        w = {k: u.clone() for k, u in v.items()}
        if name == "dt":
            w[name][b, t, h] = float(bad)
        elif name == "state":
            w[name][b, h, -1, 0] = float(bad)
        else:
            w[name][b, t, -1, -1] = float(bad)
        row = {k: u[b:b + 1] if k in ("x", "dt", "Bm", "C", "state") else u for k, u in w.items()}
        y, s = (u.cpu() for u in gpu_scan(cuda(w)))
        want, last = ref_scan(*(row[k].double() for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, row["state"].double(), None)
        for got, clean, ref in ((y, y0, want), (s, s0, last)):
            assert torch.equal(got[:b], clean[:b]) and torch.equal(got[b].isfinite(), ref[0].isfinite()), (name, t, bad)
        assert torch.equal(y[b, :t], y0[b, :t]), (name, t, bad)
        if name == "x":  # another value's outputs never take part
            assert torch.equal(y[b].flatten(1)[:, :-1], y0[b].flatten(1)[:, :-1]) and torch.equal(s[b].flatten(0, 1)[:-1], s0[b].flatten(0, 1)[:-1]), (t, bad)


def scan_gradients(v, dy, ds):
    """all gradients of a scan: the definition's and the kernels'"""
    leaves = {k: t.double().requires_grad_() for k, t in v.items()}
    out = ref_scan(*(leaves[k] for k in ("x", "dt", "A", "Bm", "C", "D", "bias")), True, leaves["state"], None)
    want = torch.autograd.grad(out, list(leaves.values()), (dy.double(), ds.double()))
    here = cuda(v, leaf=True)
    got = torch.autograd.grad(gpu_scan(here), list(here.values()), (dy.cuda(), ds.cuda()))
    return {k: (a, b) for k, a, b in zip(v, got, want)}


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sums_over_all_tokens(shape, kind):
    """gradients of A and dt_bias are sums over B L tokens (those of a head's P values are summed in each), whose magnitudes add up to at most sqrt(B L) of the result
    for random signs, an eighth of which the sums within a token have averaged out already; dt's own has no such sum"""
    B, L, H, G, P, N = shape
    v, r = scan_inputs(*shape, kind, seed=L + 1, fp32_dt=True), torch.Generator().manual_seed(2)
    far = {k: off(a, b) for k, (a, b) in scan_gradients(v, torch.randn(B, L, H, P, generator=r).to(kind), torch.randn(B, H, P, N, generator=r)).items()}
    assert max(far["A"], far["bias"]) <= tol(kind) * max(1.0, (B * L) ** 0.5 / 8) and far["dt"] <= tol(kind), far


@gpu
@pytest.mark.parametrize("A,bias", [((-2.0, -5.0), (40.0, -300.0)), ((0.05, 0.0), (0.0, 0.0)), ((-2.0, -5.0), (-60.0, -20.0))], ids=["forgets", "grows", "stands"])
def test_gradients_of_strong_and_weak_steps(A, bias):
    """states that are forgotten at once, steps that underflow to zero, states that grow or only add up, and steps whose softplus has no bits next to 1"""
    v, r = scan_inputs(2, 200, 2, 1, 16, 16, torch.float32, seed=3), torch.Generator().manual_seed(2)
    v["A"], v["bias"] = torch.tensor(A), torch.tensor(bias)
    pairs = scan_gradients(v, torch.randn(2, 200, 2, 16, generator=r), torch.randn(2, 2, 16, 16, generator=r))
    for k, (a, b) in pairs.items():
        for h in range(2) if k in ("dt", "A", "bias") else (slice(None),):  # heads apart: one has far smaller gradients
            assert off(a[..., h], b[..., h]) <= 4 * tol(torch.float32), (k, h)


@gpu
@pytest.mark.parametrize("name", ["x", "dt", "Bm", "C"])
def test_gradients_of_other_rows_keep_their_bits(name):
    v = scan_inputs(3, 700, 2, 1, 32, 32, torch.bfloat16, seed=2)
    dy = torch.randn(3, 700, 2, 32, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()

    def once(v):
        y, s = gpu_scan(v)
        return torch.autograd.grad((y, s), [v[k] for k in ("x", "dt", "Bm", "C", "state")], (dy, torch.ones_like(s)))

    w = {k: t.clone() for k, t in v.items()}
    w[name][1, 300, 0] = float("nan")
    pairs = list(zip(once(cuda(v, leaf=True)), once(cuda(w, leaf=True))))
    assert all(torch.equal(p[0], q[0]) and torch.equal(p[2], q[2]) for p, q in pairs)
    assert any(q[1].isnan().any() for _, q in pairs)
