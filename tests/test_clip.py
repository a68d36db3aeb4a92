"""rtfs_net_amd.optim.clip_grad_norm_ (csrc/clip.hip) against torch.nn.utils.clip_grad_norm_'s arithmetic in float64.

The norm is summed in fp64 and rounded once to fp32 (2 u = 1.2e-7 leaves room for the root); a scaled gradient is rounded in the factor (three fp32 operations:
the sum, the quotient, the product) and once to its own type."""
import math

import pytest
import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def params(shapes, kinds, device, seed=0, scale=1.0):
    r = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.zeros(s, dtype=kinds[i % len(kinds)], device=device))
        p.grad = (torch.randn(s, generator=r) * scale).to(p.dtype).to(device)
        out.append(p)
    return out


def check(ps, max_norm, kind):
    from rtfs_net_amd.optim import clip_grad_norm_

    before = [p.grad.clone() for p in ps]
    flat = torch.cat([g.double().flatten() for g in before])
    want = flat.abs().max() if kind == math.inf else flat.norm()
    got = clip_grad_norm_(ps, max_norm, kind)
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - float(want)) <= 2 * U[torch.float32] * float(want)
    coef = min(1.0, max_norm / (float(want) + 1e-6))
    for p, g in zip(ps, before):
        assert p.grad.shape == g.shape and p.grad.stride() == g.stride()
        err = (p.grad.double() - g.double() * coef).abs()
        tiny = torch.finfo(p.dtype).smallest_normal if p.dtype != torch.float16 else 2.0 ** -14
        assert bool((err <= (U[p.dtype] + 6 * U[torch.float32]) * g.double().abs() * coef + tiny * U[p.dtype] * 2).all())
        if coef == 1.0:
            assert torch.equal(p.grad, g)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [2.0, math.inf])
@pytest.mark.parametrize("kinds", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float32, torch.bfloat16, torch.float16]], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("shapes", [[(1,)], [(4096,), (4095,), (4097,)], [(3, 5)] * 500, [(1 << 20,), (7,), (0,), (333, 777)], [(64, 256, 1, 1), (64,)] * 120 + [(2, 3, 5, 7)]],
                         ids=["one", "units", "many", "large", "net"])
def test_clip_matches_the_formula(shapes, kinds, norm):
    check(params(shapes, kinds, "cuda"), 0.5, norm)
    check(params(shapes, kinds, "cuda", seed=1), 1e9, norm)


@pytest.mark.gpu
def test_views_at_every_alignment_and_in_every_order():
    """gradients that are slices of one flat buffer (whose neighbours stay as they are), and ones stored with their dimensions permuted"""
    from rtfs_net_amd.optim import clip_grad_norm_

    for kind in U:
        flat = torch.randn(9 * 40, device="cuda").to(kind)
        whole, ps = flat.clone(), []
        for i in range(9):
            p = torch.nn.Parameter(torch.zeros(40 - i - 1, dtype=kind, device="cuda"))
            p.grad = flat[40 * i + i:40 * i + 39]
            ps.append(p)
        check(ps, 0.25, 2.0)
        for i in range(9):
            assert torch.equal(flat[40 * i:40 * i + i], whole[40 * i:40 * i + i]) and flat[40 * i + 39] == whole[40 * i + 39]
    p = torch.nn.Parameter(torch.zeros(4, 6, 5, 5, device="cuda").to(memory_format=torch.channels_last))
    p.grad = torch.randn(4, 6, 5, 5, device="cuda").to(memory_format=torch.channels_last)
    check([p], 0.1, 2.0)
    p.grad = torch.randn(4, 6, 5, 10, device="cuda")[..., ::2]
    with pytest.raises(ValueError, match="gaps"):
        clip_grad_norm_(p, 1.0)


@pytest.mark.gpu
def test_like_torch_where_values_are_not_ordinary():
    """the largest and smallest magnitudes, infinities and NaN do what torch's clip makes of them; the same bits on every run"""
    from rtfs_net_amd.optim import clip_grad_norm_

    for values in ([1e30, -1e30], [1e-30, 0.0], [0.0, 0.0], [float("inf"), 1.0], [float("nan"), 1.0], [-float("inf"), float("nan")]):
        for norm in (2.0, math.inf):
            ps = params([(1000,), (3,)], [torch.float32], "cuda", scale=0.0)
            ps[0].grad[500], ps[1].grad[2] = values[0], values[1]
            ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in ps]
            for p, q in zip(ps, ref):
                q.grad = p.grad.double().cpu()
            want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm)
            got = clip_grad_norm_(ps, 1.0, norm)
            assert torch.allclose(got.double().cpu(), want, rtol=1e-6, atol=0.0, equal_nan=True)
            for p, q in zip(ps, ref):
                assert torch.allclose(p.grad.double().cpu(), q.grad, rtol=1e-6, atol=1e-38, equal_nan=True), (values, norm)
    a, b = params([(333, 777), (5,)] * 50, [torch.float32], "cuda"), params([(333, 777), (5,)] * 50, [torch.float32], "cuda")
    assert torch.equal(clip_grad_norm_(a, 1.0), clip_grad_norm_(b, 1.0)) and all(torch.equal(p.grad, q.grad) for p, q in zip(a, b))


@pytest.mark.gpu
def test_a_tensor_listed_twice_counts_once_and_versions_move():
    from rtfs_net_amd.optim import clip_grad_norm_

    p, q = params([(100,), (50,)], [torch.float32], "cuda")
    q.grad = None
    g, version = p.grad.clone(), p.grad._version
    norm = clip_grad_norm_((t for t in [p, p, q]), 1.0)
    assert off(norm, g.norm()) < 1e-6 and off(p.grad, g / (norm + 1e-6)) < 1e-6 and p.grad._version > version


@pytest.mark.gpu
def test_gradients_at_the_same_address_are_refused():
    from rtfs_net_amd.optim import clip_grad_norm_

    p, q, r = params([(100,), (100,), (0,)], [torch.float32], "cuda")
    empty = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    empty.grad = torch.zeros(0, device="cuda")
    clip_grad_norm_([p, q, r, empty], 1.0)
    odd = torch.nn.Parameter(torch.zeros(5, 0, device="cuda"))
    turned = torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())
    odd.grad, turned.grad = torch.zeros(5, 0, device="cuda"), torch.randn(4, 6, device="cuda").t()
    want = torch.cat([p.grad.flatten(), turned.grad.flatten()]).double().norm()
    assert off(clip_grad_norm_([p, odd, turned, r, p, empty], 0.5), want) < 1e-6
    q.grad = p.grad.view(100)
    with pytest.raises(ValueError, match="same address"):
        clip_grad_norm_([p, q, r], 1.0)


@pytest.mark.gpu
def test_more_than_2_31_elements():
    """ones, but for the ends: the norm by counting"""
    from rtfs_net_amd.optim import clip_grad_norm_

    n = (1 << 31) + 5
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    p.grad[0], p.grad[-1] = 2.0 ** 14, 2.0 ** 15
    want = math.sqrt(n - 2 + 2.0 ** 28 + 2.0 ** 30)
    norm = clip_grad_norm_(p, want / 4)
    assert abs(float(norm) / want - 1) <= 2 * U[torch.float32]
    assert float(p.grad[0]) == 2.0 ** 12 and float(p.grad[-1]) == 2.0 ** 13 and bool((p.grad[1:-1] == 0.25).all())


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.gpu
def test_captured_clip_replays():
    from rtfs_net_amd.optim import clip_grad_norm_

    ps, ref = params([(300,)] * 300, [torch.float32], "cuda"), params([(300,)] * 300, [torch.float32], "cuda")
    with torch.cuda.stream(torch.cuda.Stream()):
        clip_grad_norm_(ref, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for i in range(4):
        for p, q in zip(ps, ref):
            q.grad.normal_()
            p.grad.copy_(q.grad)
        graph.replay()
        want = clip_grad_norm_(ref, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(ps, ref)), i


def test_refusals():
    from rtfs_net_amd.optim import clip_grad_norm_

    p = params([(3,)], [torch.float32], "cpu")[0]
    for bad in (lambda: clip_grad_norm_([p], -1.0), lambda: clip_grad_norm_([p], float("nan")), lambda: clip_grad_norm_([p], 1.0, 1.0), lambda: clip_grad_norm_([p], 1.0)):
        with pytest.raises(ValueError):
            bad()
    p.grad = None
    assert float(clip_grad_norm_(p, 1.0)) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0


def test_the_library_refuses_bad_lists():
    import ctypes

    from rtfs_net_amd import lib

    h = lib.load()
    at, size, kind = (ctypes.c_longlong * 1)(4096), (ctypes.c_longlong * 1)(8), (ctypes.c_int * 1)(0)
    call = lambda at, size, kind, n, m, k, parts: h.rtfs_clip_grad_norm(at, size, kind, n, m, k, 16, parts, 16, None)  # noqa: E731
    assert call(at, size, kind, 0, 1.0, 2, 4096) == -1 and call(at, size, kind, 1, -1.0, 2, 4096) == -1 and call(at, size, kind, 1, 1.0, 1, 4096) == -1
    assert call(at, size, kind, 1, 1.0, 2, 0) == -1  # no room for the partial sums
    assert call((ctypes.c_longlong * 1)(4098), size, kind, 1, 1.0, 2, 4096) == -1  # not on an element boundary
    assert call(at, (ctypes.c_longlong * 1)(-1), kind, 1, 1.0, 2, 4096) == -1 and call(at, size, (ctypes.c_int * 1)(3), 1, 1.0, 2, 4096) == -1


def test_the_library_refuses_tensors_that_overlap():
    """before anything is launched (no device is touched): two workgroups would scale the same values at once"""
    import ctypes

    from rtfs_net_amd import lib

    h = lib.load()

    def call(*spans):  # address, size, type
        n = len(spans)
        at, size, kind = zip(*spans)
        return h.rtfs_clip_grad_norm((ctypes.c_longlong * n)(*at), (ctypes.c_longlong * n)(*size), (ctypes.c_int * n)(*kind), n, 1.0, 2, 16, 4096, 16, None)

    assert call((4096, 8, 0), (4124, 8, 0)) == -1  # the last value of the first is the first of the second
    assert call((8192, 8, 0), (4096, 8, 1), (8194, 1, 1)) == -1 and call((4096, 100, 1), (4098, 1, 1), (8192, 1, 0)) == -1
    assert call((4096, 8, 0), (0, 0, 0), (4096, 8, 0)) == -1


@pytest.mark.gpu
def test_gradients_that_overlap_are_refused():
    from rtfs_net_amd.optim import clip_grad_norm_

    flat = torch.randn(300, device="cuda")
    held = flat.clone()
    ps = params([(100,), (100,), (50,), (0,)], [torch.float32], "cuda")
    ps[0].grad, ps[1].grad = flat[150:250], flat[51:151]
    with pytest.raises(ValueError, match="memory in common"):
        clip_grad_norm_(ps, 0.1)
    assert torch.equal(flat, held)
    ps[1].grad = flat[50:150]
    check(ps, 0.1, 2.0)
    assert torch.equal(flat[:50], held[:50]) and torch.equal(flat[250:], held[250:])


def split_params(total, count):
    flat, ps = torch.randn(total, device="cuda").bfloat16(), []
    for g in flat.split(total // count):
        p = torch.nn.Parameter(g.detach())
        p.grad = g
        ps.append(p)
    return ps


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [2.0, math.inf])
def test_lists_of_thousands(norm):
    """so many launches that their partial sums are added up by one of their own"""
    check(params([(n,) for n in range(8193, 8193 + 2900)], list(U), "cuda"), 0.5, norm)
    check(params([(3,)] * 5000, [torch.float32], "cuda"), 0.5, norm)


@pytest.mark.gpu
def test_a_long_list_keeps_the_card_busy():
    """the same values in 20 times as many tensors: 21 launches instead of one each way, and not the time of a card that stands mostly empty"""
    from rtfs_net_amd.optim import clip_grad_norm_

    times = []
    for count in (240, 5000):
        ps = split_params(240_000_000, count)
        clip_grad_norm_(ps, 1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            clip_grad_norm_(ps, 1.0)
        best = math.inf
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] < 3 * times[0], times


@pytest.mark.gpu
def test_captured_long_list_replays():
    from rtfs_net_amd.optim import clip_grad_norm_

    a, b = (split_params(24_000_007, 2500) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(a, 1.0)
    for i in range(4):
        for p, q in zip(a, b):
            q.grad.normal_()
            p.grad.copy_(q.grad)
        graph.replay()
        want = clip_grad_norm_(b, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(a, b)), i
