"""clip_grads_ / clip_grad_norm_ / LoRAGradReducer.reduce(max_norm) against float64 and torch.nn.utils.clip_grad_norm_.

The squares are exact products of fp32 values in fp64, so the norm is good to its own rounding (2^-24) plus the fp64 sum's; the factor is
rounded once to fp32 and every product once to fp32 and once to the output's type: 3 * 2^-24 + u of the value, u = 2^-8 for bf16."""
import math

import pytest
import torch

from image_segmentation_amd import _C, LoRAGradReducer, clip_grad_norm_, clip_grads_

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def make(sizes, kinds, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * (1 + i % 3)).to("cuda", k) for i, (n, k) in enumerate(zip(sizes, kinds))]


def total(grads, p=2.0):
    if p == math.inf:
        return max(float(g.double().abs().max()) for g in grads if g.numel())
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check_scaled(got, src, factor):
    for a, s in zip(got, src):
        want = s.double() * factor
        u = 2.0 ** -8 if a.dtype == BF else 0.0
        assert ((a.double() - want).abs() <= (4 * E + u) * want.abs() + 1e-38).all()


SETS = [([1], [FP]), ([1], [BF]), ([0, 3, 0], [FP, BF, FP]), ([7, 8, 9, 2047, 2048, 2049], [BF] * 6), ([5000, 1, 70000, 333], [FP, BF, BF, FP]),
        ([17 + 5 * i for i in range(300)], [FP if i % 2 else BF for i in range(300)]), ([3_000_001, 12, 1_500_000], [BF, FP, FP]),
        ([9_000_001], [FP])]


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("sizes, kinds", SETS)
@pytest.mark.parametrize("form", ["place", "fp32", "bf16", "same"])
def test_matches_float64(sizes, kinds, form, p):
    grads = make(sizes, kinds, sum(sizes))
    src = [g.clone() for g in grads]
    want = total(src, p)
    out = {"place": None, "fp32": [torch.full_like(g, float("nan"), dtype=FP) for g in grads],
           "bf16": [torch.full_like(g, float("nan"), dtype=BF) for g in grads], "same": [torch.empty_like(g) for g in grads]}[form]
    for limit in (0.37 * want, 3.0 * want):
        for g, s in zip(grads, src):
            g.copy_(s)
        norm = clip_grads_(grads, limit, p, out=out)
        assert norm.dtype == FP and norm.shape == () and abs(float(norm) - want) <= 2 * E * want
        check_scaled(grads if out is None else out, src, min(1.0, limit / (want + 1e-6)))
        if out is not None or limit > want:
            assert all(torch.equal(g, s) for g, s in zip(grads, src))         # the inputs, and gradients below the limit, are untouched
    norm = clip_grads_(src, math.inf, p)
    assert abs(float(norm) - want) <= 2 * E * want and all(torch.equal(g, s) for g, s in zip(src, make(sizes, kinds, sum(sizes))))


def test_some_in_place():
    # outputs that are their own inputs beside others that are not, over more tensors than a launch takes
    grads = make([40 + i for i in range(230)], [BF if i % 3 == 0 else FP for i in range(230)], 31)
    src = [g.clone() for g in grads]
    out = [g if i % 2 else torch.empty_like(g, dtype=FP) for i, g in enumerate(grads)]
    want = total(src)
    for limit in (2.0 * want, 0.5 * want):
        clip_grads_(grads, limit, out=out)
        check_scaled(out, src, min(1.0, limit / (want + 1e-6)))
        assert all(torch.equal(g, s) for i, (g, s) in enumerate(zip(grads, src)) if i % 2 == 0 or limit > want)


@pytest.mark.parametrize("kind", [FP, BF])
def test_alignment(kind):
    # views that begin anywhere in one buffer, with guards between them
    sizes = [1, 5, 2049, 16, 7, 4096, 33, 3]
    flat = torch.full((sum(sizes) + 3 * len(sizes) + 3,), 7.0, dtype=kind, device="cuda")
    out_flat = torch.full((flat.numel() + 1,), 7.0, device="cuda")
    views, outs, o = [], [], 1
    for n in sizes:
        views.append(flat[o:o + n])
        outs.append(out_flat[o + 1:o + 1 + n])
        o += n + 3
    src = make(sizes, [kind] * len(sizes), 5)
    for v, s in zip(views, src):
        v.copy_(s)
    want = total(src)
    clip_grads_(views, 0.5 * want, out=outs)
    check_scaled(outs, src, 0.5 * want / (want + 1e-6))
    clip_grads_(views, 0.5 * want)
    check_scaled(views, src, 0.5 * want / (want + 1e-6))
    for buf, off in ((flat, 0), (out_flat, 1)):
        guard = torch.ones_like(buf, dtype=torch.bool)
        o = 1
        for n in sizes:
            guard[o + off:o + off + n] = False
            o += n + 3
        assert (buf[guard] == 7.0).all()


def test_range_and_zeros():
    for s in (1e-30, 1e25):                                   # squares far outside fp32
        g = make([1000, 64], [FP, FP], 3, s)
        want = total(g)
        assert abs(float(clip_grads_(g, math.inf)) - want) <= 2 * E * want
    z = [torch.zeros(100, device="cuda"), torch.zeros(5, device="cuda", dtype=BF)]
    assert float(clip_grads_(z, 1.0)) == 0.0 and all((t == 0).all() for t in z)
    g = make([50], [FP], 4)
    clip_grads_(g, 0.0)
    assert (g[0] == 0).all()
    assert float(clip_grads_([torch.empty(0, device="cuda")], 1.0)) == 0.0
    assert float(clip_grads_([], 1.0)) == 0.0
    g = make([100], [FP], 6)
    want = total(g)
    s = g[0].clone()
    assert abs(float(clip_grads_(g, 0.25 * want, grad_scale=-0.5)) - 0.5 * want) <= 2 * E * want
    check_scaled(g, [s], -0.5 * 0.25 * want / (0.5 * want + 1e-6))


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_not_finite(bad, p):
    grads = make([300, 40], [FP, BF], 7)
    grads[1][3] = bad
    src = [g.clone() for g in grads]
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grads_(grads, 1.0, p, error_if_nonfinite=True)
    assert all(torch.equal(g.nan_to_num(), s.nan_to_num()) for g, s in zip(grads, src))
    norm = clip_grads_(grads, 1.0, p)
    params = [torch.nn.Parameter(torch.zeros_like(s)) for s in src]
    for q, s in zip(params, src):
        q.grad = s.clone()
    ref = torch.nn.utils.clip_grad_norm_(params, 1.0, p)
    assert float(norm) == float(ref) or (norm.isnan() and ref.isnan())
    for g, q in zip(grads, params):
        assert torch.allclose(g, q.grad, rtol=0, atol=0, equal_nan=True)


def test_parameters_like_torch():
    torch.manual_seed(0)
    shapes = [(64, 32), (64,), (7, 3, 5, 5), (1,), (130, 257)]
    a = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    for q in a:
        q.grad = torch.randn_like(q)
    a[2].grad = a[2].grad.contiguous(memory_format=torch.channels_last)       # another layout than the parameter's
    a[4].grad = torch.randn(257, 130, device="cuda").t()
    a.append(torch.nn.Parameter(torch.zeros(4, device="cuda")))                # no gradient
    b = [torch.nn.Parameter(q.detach().clone()) for q in a]
    for q, r in zip(a, b):
        r.grad = None if q.grad is None else q.grad.clone()
    v = a[0].grad._version
    n1 = clip_grad_norm_(iter(a + [a[0]]), 2.5)                                # a parameter listed twice counts once
    n2 = torch.nn.utils.clip_grad_norm_(b, 2.5)
    assert abs(float(n1) - float(n2)) <= 1e-6 * float(n2)                      # torch sums in fp32
    assert a[0].grad._version > v
    for q, r in zip(a, b):
        assert q.grad is r.grad is None or (q.grad - r.grad).abs().max() <= 2e-6 * r.grad.abs().max()
    single = torch.nn.Parameter(torch.ones(3, device="cuda"))
    single.grad = torch.full((3,), 2.0, device="cuda")
    assert abs(float(clip_grad_norm_(single, 1.0)) - 12 ** 0.5) < 1e-6


def test_refusals():
    g = make([64], [FP], 1)[0]
    for bad, kw in (([g.half()], {}), ([g.double()], {}), ([g, g], {}), ([g[:40], g[30:]], {}), ([g, g.cpu()], {}), ([g.long()], {}),
                    ([g[:32], g[32:]], dict(out=[g[32:], g[:32]])), ([g[:32]], dict(out=[g[1:33]])), ([g], dict(out=[g.half()])), ([g], dict(norm_type=3))):
        with pytest.raises(_C.LsamError):
            clip_grads_(bad, 1.0, **kw)
    assert float(clip_grads_([g, g], math.inf)) > 0           # the norm alone may take a tensor twice


def test_same_bits_stream_graph():
    sizes, kinds = [40_000, 7, 130_001, 5000], [FP, BF, BF, FP]
    grads = make(sizes, kinds, 9)
    out = [torch.empty_like(g, dtype=FP) for g in grads]
    limit = 0.2 * total(grads)
    n0 = clip_grads_(grads, limit, out=out)
    want = [o.clone() for o in out]
    assert torch.equal(clip_grads_(grads, limit, out=out), n0) and all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(clip_grads_(grads, limit, out=out), n0) and all(torch.equal(a, b) for a, b in zip(out, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = clip_grads_(grads, limit, out=out)
    for seed in (11, 13, 17):
        fresh = make(sizes, kinds, seed, 0.1 * (seed - 10))
        for g, f in zip(grads, fresh):
            g.copy_(f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = [torch.empty_like(o) for o in out]
        assert torch.equal(norm, clip_grads_(fresh, limit, out=ref)) and all(torch.equal(a, b) for a, b in zip(out, ref))


def test_reducer_clips_the_mean(tmp_path):
    """reduce(max_norm): without a process group the gradients are clipped in place; on a one-rank group the flat buffer is clipped
    into .grad, missing gradients counting as zero.  (gloo takes CPU tensors only; RCCL serves the one-rank group.)"""
    import torch.distributed as dist
    params = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (300, 41, 8, 1000, 5)]
    grads = make([300, 41, 8, 1000, 5], [FP] * 5, 21)
    red = LoRAGradReducer(params)

    def fill(skip=None):
        for i, (p, g) in enumerate(zip(params, grads)):
            p.grad = None if i == skip else g.clone()

    fill()
    want = total(grads)
    assert red.reduce() is None and all(torch.equal(p.grad, g) for p, g in zip(params, grads))
    n = red.reduce(max_norm=0.3 * want)
    assert abs(float(n) - want) <= 2 * E * want
    check_scaled([p.grad for p in params], grads, 0.3 * want / (want + 1e-6))
    assert not dist.is_initialized()
    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        red = LoRAGradReducer(params)
        fill(skip=2)
        src = [torch.zeros_like(g) if i == 2 else g for i, g in enumerate(grads)]
        want = total(src)
        n = red.reduce(max_norm=0.3 * want)
        assert abs(float(n) - want) <= 2 * E * want
        check_scaled([p.grad for p in params], src, 0.3 * want / (want + 1e-6))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("kw", [{}, dict(error_if_nonfinite=True)])
def test_norm_alone_writes_nothing(kw):
    # tensors of any layout, expanded ones and ones that share memory among them: read, and neither written nor marked as written
    base = make([24, 6, 5], [FP, BF, FP], 41)
    grads = [base[0].view(4, 6).t(), base[0].view(4, 6), base[1].expand(3, 6), base[2][::2]]
    want = total(grads)
    versions = [g._version for g in base]
    norm = clip_grads_(grads, math.inf, **kw)
    assert abs(float(norm) - want) <= 2 * E * want
    assert versions == [g._version for g in base] and all(torch.equal(g, s) for g, s in zip(base, make([24, 6, 5], [FP, BF, FP], 41)))
    # what is saved for a backward stays good
    x = torch.ones(2, 3, device="cuda").t().clone(memory_format=torch.preserve_format).requires_grad_(True)
    y = x * 2
    z = y * y
    clip_grads_([y.detach()], math.inf)
    z.sum().backward()
    assert (x.grad == 8).all()


def test_reducer_refuses_types_before_the_exchange(tmp_path):
    # a gradient that cannot be clipped is refused while every rank's buckets are as they were, not behind the exchange
    import torch.distributed as dist
    params = [torch.nn.Parameter(torch.zeros(5, device="cuda")), torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float16))]
    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        red = LoRAGradReducer(params)
        for p in params:
            p.grad = torch.ones_like(p)
        with pytest.raises(_C.LsamError, match="float16"):
            red.reduce(max_norm=1.0)
        assert red.stats["all_reduce"] == 0 and all((p.grad == 1).all() for p in params)
        red.reduce()
        assert red.stats["all_reduce"] == 1 and all((p.grad == 1).all() for p in params)
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("n", [2 ** 30 + 7, 2 ** 32 + 5])
def test_a_tensor_of_more_than_2_to_30_values(n):
    g = torch.full((n,), 0.5, dtype=BF, device="cuda")
    g[-3:] = 64.0
    want = math.sqrt((n - 3) * 0.25 + 3 * 4096.0)
    norm = clip_grads_([g], want / 4)
    assert abs(float(norm) - want) <= 2 * E * want
    assert (g[:-3] == 0.125).all() and (g[-3:] == 16.0).all()   # a quarter, less 1e-6 of the norm: the nearest bf16 value
    assert abs(float(clip_grads_([g], math.inf, math.inf)) - 16.0) == 0.0
