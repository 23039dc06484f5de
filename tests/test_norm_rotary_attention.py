"""Layer norm, rotary positions and 16-bit cross attention: what can be checked without a GPU (frequencies, refusals of the C
entry points, of CPU tensors), and on a GPU a training step through all of them together and through the Attention module."""
import math

import pytest
import torch

from q8_kernels_amd import _lib, functional as Q8F
from q8_kernels_amd.functional.rotary import apply_rotary, rotary_frequencies

BF16 = torch.bfloat16


def test_frequencies():
    f, factor = rotary_frequencies(8)
    assert f.dtype == torch.float64 and factor == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    lin, one = rotary_frequencies(8, scaling="linear", stretch=4.0)
    assert torch.equal(lin, f / 4.0) and one == 1.0
    ntk, _ = rotary_frequencies(8, scaling="ntk", stretch=4.0)          # the fastest pair stays, the slowest is interpolated
    assert ntk[0] == f[0] and math.isclose(float(ntk[-1]), float(f[-1]) / 4.0, rel_tol=1e-12)
    yarn, factor = rotary_frequencies(128, scaling="by_parts", stretch=16.0, trained_positions=4096)
    plain, _ = rotary_frequencies(128)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32]) and torch.equal(yarn[turns <= 1], plain[turns <= 1] / 16.0)
    between = (turns > 1) & (turns < 32)
    assert bool(between.any()) and bool(((yarn < plain) & (yarn > plain / 16.0))[between].all())
    assert math.isclose(factor, 0.1 * math.log(16.0) + 1.0)
    assert torch.equal(rotary_frequencies(128, scaling="by_parts")[0], plain)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, stretch=0.5), dict(rotary_dim=2, scaling="ntk"),
                dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, scaling="by_parts", low_turns=3.0, high_turns=3.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 2, 4, 64, dtype=BF16)
    f = rotary_frequencies(64)[0]
    for call in (lambda: Q8F.layer_norm.layer_norm(x), lambda: apply_rotary(x, None, None, f), lambda: Q8F.cross_attention.cross_attention(x, x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_refusals_of_the_c_entry_points():
    L, (B16, F16, F32, E4) = _lib.lib(), (_lib.Q8_BF16, _lib.Q8_F16, _lib.Q8_F32, _lib.Q8_E4M3)
    ln = lambda x=16, dt=B16, st=64, w=None, b=None, wd=F32, y=16, m=None, r=None, rows=4, dim=64, eps=1e-5: (  # noqa: E731
        L.q8_layernorm(x, dt, st, w, b, wd, y, m, r, rows, dim, eps, None))
    assert ln(rows=0, x=None, y=None) == 0
    assert ln(x=None) == -1 and ln(y=None) == -1 and ln(m=16) == -1
    assert ln(dt=E4) == -2 and ln(w=16, wd=F16) == -2
    assert ln(dim=0) == -3 and ln(dim=32769) == -3 and ln(rows=-1) == -3 and ln(rows=1 << 32) == -3 and ln(st=63) == -3 and ln(eps=-1.0) == -3
    assert ln(x=17) == -4 and ln(w=18) == -4
    assert L.q8_layernorm_backward_workspace(100, 64) > 0 and L.q8_layernorm_backward_workspace(-1, 64) == -3 and L.q8_layernorm_backward_workspace((1 << 63) - 1, 64) == -3
    lb = lambda g=16, x=16, dt=B16, w=None, m=16, r=16, dx=16, dw=None, db=None, ws=None, size=0, rows=4, dim=64: (  # noqa: E731
        L.q8_layernorm_backward(g, dim, x, dt, dim, w, F32, m, r, dx, dw, db, ws, size, rows, dim, None))
    assert lb(dx=None) == 0 and lb(rows=0, g=None, x=None, m=None, r=None) == 0
    assert lb(g=None) == -1 and lb(m=None) == -1 and lb(dw=16) == -1
    assert lb(dw=16, ws=16, size=8) == -3 and lb(dx=17) == -4 and lb(dt=E4) == -2
    st = _lib._i64 * 3
    ok, neg, big, odd = st(4096, 512, 64), st(-64, 512, 64), st(1 << 62, 512, 64), st(4096, 512, 60)

    def rot(q=16, qs=ok, qo=16, qos=ok, h=8, k=None, ks=None, ko=None, kos=None, hk=0, dt=B16, p=None, bits=0, row=0, f=16, r=64, b=2, t=8, d=64):
        return L.q8_rotary(q, qs, qo, qos, h, k, ks, ko, kos, hk, dt, p, bits, row, f, r, 1, 1.0, 0, b, t, d, None)

    assert rot(b=0, q=None, qs=None) == 0 and rot(h=0, q=None) == 0
    assert rot(q=None) == -1 and rot(qs=None) == -1 and rot(f=None) == -1 and rot(hk=2) == -1
    assert rot(dt=E4) == -2 and rot(p=16, bits=16) == -2
    assert rot(r=63) == -3 and rot(r=0) == -3 and rot(r=66) == -3 and rot(d=513) == -3 and rot(qs=neg) == -3 and rot(qs=big) == -3 and rot(b=-1) == -3
    assert rot(p=16, bits=64, row=4) == -3 and rot(b=1 << 40, t=1 << 40) == -3
    assert rot(q=17) == -4 and rot(f=20) == -4 and rot(p=20, bits=64) == -4

    def att(q=16, qs=ok, k=16, v=16, o=16, os=ok, lse=None, lens=None, mask=None, mrow=0, dt=B16, scale=0.1, b=2, h=8, hk=8, m=8, n=8, d=64, ws=None, size=0):
        return L.q8_cross_attn(q, qs, k, ok, v, ok, o, os, lse, lens, mask, mrow, dt, scale, b, h, hk, m, n, d, ws, size, None)

    assert att(b=0, q=None) == 0 and att(m=0, q=None, o=None) == 0
    assert att(q=None) == -1 and att(k=None) == -1 and att(o=None) == -1 and att(os=None) == -1
    assert att(dt=F32) == -2 and att(dt=E4) == -2
    assert att(h=8, hk=3) == -3 and att(d=60) == -3 and att(d=136) == -3 and att(n=-1) == -3 and att(scale=0.0) == -3 and att(scale=float("nan")) == -3
    assert att(scale=float("inf")) == -3 and att(qs=neg) == -3 and att(qs=st(4096, 512, 1 << 24)) == -3 and att(mask=16, mrow=-1) == -3
    assert att(q=24) == -4 and att(qs=odd) == -4 and att(lens=17) == -4
    need = L.q8_cross_attn_workspace(2, 8, 8, 8, 100000, 64)
    assert need > 0 and att(n=100000) == -1 and att(n=100000, ws=16, size=16) == -3
    assert L.q8_cross_attn_workspace(2, 8, 3, 8, 8, 64) == -3 and L.q8_cross_attn_backward_workspace(2, 8, 8, 8, 8, 60) == -3

    def bwd(g=16, lse=16, dq=16, dk=16, ws=16, size=1 << 40, dt=B16, d=64, n=300, qs=ok, b=2, h=8):
        return L.q8_cross_attn_backward(g, ok, 16, qs, 16, ok, 16, ok, 16, ok, lse, dq, ok, dk, ok, 16, ok, None, None, 0, dt, 0.1, b, h, h, 8, n, d, ws, size, None)

    assert bwd(g=None) == -1 and bwd(lse=None) == -1 and bwd(dq=None) == -1 and bwd(dk=None) == -1 and bwd(ws=None) == -1
    assert bwd(size=16) == -3 and bwd(d=12) == -3 and bwd(dt=F32) == -2 and bwd(ws=20) == -4 and bwd(qs=odd) == -4
    # more workgroups than a launch takes (2^32 threads)
    assert ln(rows=(1 << 31) - 1) == -3 and ln(rows=1 << 25, dim=8000, st=8000) == -3 and ln(rows=1 << 23, dim=9000, st=9000) == -3
    assert rot(h=1, b=1, t=1 << 34, d=8, r=8) == -3
    assert att(b=1 << 20, h=16, hk=16, m=1) == -3 and att(b=1 << 16, h=1 << 12, hk=1, n=300) == -3
    assert bwd(b=1 << 20, h=16) == -3 and bwd(b=1 << 20, h=16, n=8) == -3


@pytest.mark.gpu
def test_together_with_gradients(dev):
    """norm -> projections -> rotary -> attention and back. Each operator is checked against its definition in float64 on the
    inputs and the upstream gradients that it really had, with the tolerances of its own tests."""
    import test_cross_attention_gpu as A
    import test_layer_norm_gpu as N
    import test_rotary_gpu as R
    gen = torch.Generator(device=dev).manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    b, t, s, h, hk, d, dim = 2, 37, 53, 8, 2, 64, 512
    x, text = rnd(b, t, dim).to(BF16).requires_grad_(), rnd(b, s, dim).to(BF16).requires_grad_()
    w, bias = (1 + 0.1 * rnd(dim)).requires_grad_(), (0.1 * rnd(dim)).requires_grad_()
    wq, wk, wv = ((rnd(dim, n * d) * dim ** -0.5).to(BF16).requires_grad_() for n in (h, hk, hk))
    f = rotary_frequencies(32)[0].to(dev)
    lens = torch.tensor([s, 20], dtype=torch.int32, device=dev)
    split = lambda y, n: y.view(b, -1, n, d).transpose(1, 2)  # noqa: E731
    y = Q8F.layer_norm.layer_norm(x, w, bias)
    q, k, v = split(y @ wq, h), split(text @ wk, hk), split(text @ wv, hk)
    pq, pk = torch.arange(t, device=dev), torch.arange(s, device=dev)
    rq, rk = apply_rotary(q, None, pq, f), apply_rotary(k, None, pk, f)
    o = Q8F.cross_attention.cross_attention(rq, rk, v, kv_lens=lens)
    go = rnd(*o.shape).to(BF16)
    names = "o rq rk v q k y x w bias text wq wk wv".split()
    given = (o, rq, rk, v, q, k, y, x, w, bias, text, wq, wk, wv)
    g = dict(zip(names, torch.autograd.grad(o, given, go)))
    assert all(bool(torch.isfinite(z).all()) for z in g.values())
    (ny, ndx, ndw, ndb), tol = N.reference(x.detach().reshape(-1, dim), w.detach(), bias.detach(), g["y"].reshape(-1, dim), 1e-5)
    for got, want, e in ((y, ny, tol[0]), (g["x"], ndx, tol[1]), (g["w"], ndw, tol[2]), (g["bias"], ndb, tol[3])):
        assert ((got.detach().double().reshape(want.shape) - want).abs() <= e + N.half_step(want, got.dtype) + N.half_step(e, got.dtype)).all()
    for out, src, pos, gout, gin in ((rq, q, pq, g["rq"], g["q"]), (rk, k, pk, g["rk"], g["k"])):
        R.close(out.detach(), R.rotated(src.detach(), pos, f, "half", 1.0), "rotary")
        R.close(gin, R.rotated(gout, pos, f, "half", 1.0, -1), "rotary's gradient")
    valid = torch.arange(s, device=dev) < lens[:, None]
    want, tol = A.reference(rq.detach(), rk.detach(), v.detach(), go, d ** -0.5, valid)
    for name, got, r, e in zip(("o", "dq", "dk", "dv"), (o.detach(), g["rq"], g["rk"], g["v"]), want, tol):
        A.close(got, r, e, name)


@pytest.mark.gpu
def test_attention_module_runs_the_16_bit_kernels(dev, monkeypatch):
    from q8_kernels_amd.modules import Attention, Q8LinearLora
    from q8_kernels_amd.modules import attention as module
    torch.manual_seed(0)
    attn = Attention(256, 4, 64, bias=True, out_bias=True, qk_rms_norm=True).to(dev)
    for name in ("to_q", "to_k", "to_v", "to_out"):
        layer = Q8LinearLora.from_linear(torch.nn.Linear(256, 256, device=dev, dtype=BF16), r=8)
        with torch.no_grad():
            layer.lora_b.normal_(std=0.05)
        setattr(attn, name, layer)
    seen = []
    kernel = module.Q8F.cross_attention.cross_attention

    def watched(q, k, v, softmax_scale=None, kv_lens=None, key_mask=None):
        out = kernel(q, k, v, softmax_scale, kv_lens, key_mask)
        seen.append((q, k, v, kv_lens, key_mask, out))
        return out

    monkeypatch.setattr(module.Q8F.cross_attention, "cross_attention", watched)
    x, text = torch.randn(2, 30, 256, device=dev, dtype=BF16), torch.randn(2, 50, 256, device=dev, dtype=BF16)
    lens = torch.tensor([50, 17], device=dev)
    kw = dict(mm_out_dtype=BF16, attn_type="16bit", encoder_hidden_states=text)
    a = attn(x, attention_mask=lens, **kw)
    mask = torch.arange(50, device=dev) < lens[:, None]
    b = attn(x, attention_mask=mask.int(), **kw)
    assert torch.equal(a, b) and len(seen) == 2 and seen[0][3].dtype == torch.int32 and seen[1][4].dtype == torch.bool
    q, k, v, _, _, out = seen[0]
    import test_cross_attention_gpu as A
    want, tol = A.reference(q.detach(), k.detach(), v.detach(), torch.zeros_like(q), 0.125, mask)
    A.close(out.detach(), want[0], tol[0], "o")
    assert torch.equal(a, attn.to_out(out.transpose(1, 2).reshape(2, 30, 256), out_dtype=BF16))
    a.float().square().mean().backward()
    for name in ("to_q", "to_k", "to_v", "to_out"):
        layer = getattr(attn, name)
        assert all(bool(torch.isfinite(p.grad).all()) and bool((p.grad != 0).any()) for p in (layer.lora_a, layer.lora_b))
    # the same with torch's attention: what differs is the roundings of o, seen through a loss that is smooth in them
    with torch.no_grad():
        t = attn(x, attention_mask=lens, mm_out_dtype=BF16, attn_type="torch", encoder_hidden_states=text)
    assert torch.nn.functional.cosine_similarity(a.float().flatten(), t.float().flatten(), dim=0) > 0.999
    with pytest.raises(ValueError):
        attn(x, attn_type="other", mm_out_dtype=BF16)


def leaves_and_step(dev):
    """The three operators in a row, on leaves of their own, and their gradients."""
    gen = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    x, q = rnd(2, 70, 256).to(BF16), rnd(2, 4, 70, 64).to(BF16)
    w, v = 1 + 0.1 * rnd(256), rnd(2, 4, 70, 64).to(BF16)
    grad, f = rnd(2, 4, 70, 64).to(BF16), rotary_frequencies(64)[0].to(dev)

    def step(x, q, v, w):
        k = Q8F.layer_norm.layer_norm(x, w).view(2, 70, 4, 64).transpose(1, 2)
        rq, rk = apply_rotary(q, k, None, f)
        return Q8F.cross_attention.cross_attention(rq, rk, v)

    return [t.requires_grad_() for t in (x, q, v, w)], grad, step


@pytest.mark.gpu
def test_captured_training_step(dev):
    leaves, grad, step = leaves_and_step(dev)

    def eager():
        o = step(*leaves)
        return (o.detach(),) + torch.autograd.grad(o, leaves, grad)

    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(*leaves)
        out = (o.detach(),) + torch.autograd.grad(o, leaves, grad)
    del o
    for turn in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.75).add_(0.01 * turn)
        graph.replay()
        want = eager()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_is_refused(dev):
    (x, q, v, w), _, step = leaves_and_step(dev)
    f = rotary_frequencies(64)[0].to(dev)
    alive = step(x, q, v, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: Q8F.layer_norm.layer_norm(x), lambda: Q8F.layer_norm.layer_norm(x.detach(), w), lambda: apply_rotary(q, None, None, f),
                     lambda: Q8F.cross_attention.cross_attention(q.detach(), q.detach(), v)):
            with pytest.raises(RuntimeError, match="eager graph"):
                call()
        with torch.no_grad():
            o = step(x, q, v, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, alive.detach())
    with pytest.raises(RuntimeError, match="inv_freq"):
        apply_rotary(q, None, None, f.clone().requires_grad_())


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """The same training step on two streams, calls of both under way together, against one after the other."""
    leaves, grad, step = leaves_and_step(dev)
    other = [(0.5 * t.detach() + 0.25).requires_grad_() for t in leaves]

    def run(x):
        o = step(*x)
        return (o.detach(),) + torch.autograd.grad(o, x, grad)

    want = [run(leaves), run(other)]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate((leaves, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


@pytest.mark.gpu
def test_norm_and_rotary_rows_beyond_32_bits(dev):
    far = torch.empty(300 * 2 ** 23, dtype=BF16, device=dev).as_strided((300, 512), (2 ** 23, 1))
    x = torch.randn(300, 512, device=dev).to(BF16)
    far.copy_(x)
    assert torch.equal(Q8F.layer_norm.layer_norm(far), Q8F.layer_norm.layer_norm(x))
    q, f = far.view(1, 300, 8, 64).transpose(1, 2), rotary_frequencies(64)[0].to(dev)
    assert torch.equal(apply_rotary(q, None, None, f), apply_rotary(x.view(1, 300, 8, 64).transpose(1, 2), None, None, f))


@pytest.mark.gpu
def test_forms_of_the_calls(dev):
    """Arguments that mean the same give the same bits: one and many dimensions, views, one tensor in two places, parts that need no gradient."""
    gen = torch.Generator(device=dev).manual_seed(5)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    norm, attend = Q8F.layer_norm.layer_norm, Q8F.cross_attention.cross_attention
    x, w, b = rnd(3, 4, 5, 72).to(BF16), 1 + 0.1 * rnd(72), rnd(72)
    flat = norm(x.reshape(60, 72), w, b)
    assert torch.equal(norm(x, w, b).reshape(60, 72), flat) and torch.equal(norm(x[1, 2, 3], w, b), flat[33])
    assert torch.equal(norm(x.transpose(0, 2), w, b).transpose(0, 2).reshape(60, 72), flat)
    assert torch.equal(norm(x.reshape(60, 72), torch.stack((w, w), 1)[:, 0], b), flat)
    one = x[0, 0, 0].clone().requires_grad_()
    wg = w.clone().requires_grad_()
    g = rnd(72).to(BF16)
    d1, dw = torch.autograd.grad(norm(one, wg, b), (one, wg), g)
    d2 = torch.autograd.grad(norm(x[0, 0, 0], wg, b), wg, g)[0]
    assert d1.shape == (72,) and torch.equal(dw, d2)

    q, k, v = (rnd(2, n, h, 64).to(BF16).transpose(1, 2) for n, h in ((40, 8), (70, 2), (70, 2)))
    lens, mask, go = torch.tensor([70, 33], dtype=torch.int32, device=dev), rnd(2, 70) > -1, rnd(2, 8, 40, 64).to(BF16)
    want = attend(q, k, v, None, lens, mask)
    assert torch.equal(attend(q, k, v, 0.125, torch.stack((lens, lens), 1)[:, 0], mask.t().contiguous().t()), want)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    every = torch.autograd.grad(attend(*leaves, None, lens, mask), leaves, go)
    for i in range(3):
        args = [leaves[j] if j == i else leaves[j].detach() for j in range(3)]
        assert torch.equal(torch.autograd.grad(attend(*args, None, lens, mask), leaves[i], go)[0], every[i])
    both = torch.autograd.grad(attend(leaves[0], leaves[1], leaves[1], None, lens, mask), leaves[1], go)[0]
    twice = [leaves[1].detach().requires_grad_() for _ in range(2)]
    apart = torch.autograd.grad(attend(leaves[0], *twice, None, lens, mask), twice, go)
    assert torch.equal(both, apart[0] + apart[1])
    # a shared key head is the same as its copies, gradients summed
    wide = [leaves[0]] + [t.detach().repeat_interleave(4, 1).requires_grad_() for t in leaves[1:]]
    o = attend(*wide, None, lens, mask)
    assert torch.equal(o, want)
    copies = torch.autograd.grad(o, wide, go)
    assert torch.equal(copies[0], every[0])
    for a, c in zip(every[1:], copies[1:]):
        c = c.double().view(2, 2, 4, 70, 64)
        # each copy is rounded once, and the shared one too; P and dS are the same
        assert ((a.double() - c.sum(2)).abs() <= 2.0 ** -8 * (a.double().abs() + c.abs().sum(2)) + 1e-5).all()

    f, positions = rotary_frequencies(64)[0].to(dev), torch.randint(0, 9999, (2, 40), generator=gen, device=dev)
    turned = apply_rotary(q, None, positions, f)
    assert torch.equal(apply_rotary(q, None, positions.t().contiguous().t().int(), f), turned)
    assert torch.equal(apply_rotary(q[:1], None, positions[:1], f), turned[:1]) and torch.equal(apply_rotary(q[:1], None, positions[0], f), turned[:1])
    assert torch.equal(apply_rotary(q, q, positions, f)[1], turned)


@pytest.mark.gpu
def test_attention_module_self_attention_with_positions(dev):
    from q8_kernels_amd.modules import Attention, Q8Linear
    torch.manual_seed(1)
    attn = Attention(256, 4, 64, bias=True, out_bias=True, qk_rms_norm=True, use_rope=True).to(dev)
    for name in ("to_q", "to_k", "to_v", "to_out"):
        setattr(attn, name, Q8Linear.from_linear(torch.nn.Linear(256, 256, device=dev, dtype=BF16)))
    x = torch.randn(2, 60, 256, device=dev, dtype=BF16)
    angle = torch.rand(2, 60, 128, device=dev).repeat_interleave(2, -1) * 6
    with torch.no_grad():
        a, t = (attn(x, freqs_cis=(angle.cos(), angle.sin()), mm_out_dtype=BF16, attn_type=kind) for kind in ("16bit", "torch"))
    assert torch.nn.functional.cosine_similarity(a.float().flatten(), t.float().flatten(), dim=0) > 0.999
