"""Token-sequence operators (scaled embedding with its gradient by sorted tokens, causal convolution, selective scan,
gradient clipping): restatements in float64 against autograd and differences and the refusals on the CPU, the HIP kernels
against the restatements on the GPU.

Bounds: a result that is rounded to type t is off by at most half a step, u(t) = finfo(t).eps / 2, of itself; fp32 arithmetic
adds c * 2^-24 of the sum of its terms' magnitudes, c the number of roundings on the longest path (given at each use)."""
import ctypes
import math

import pytest
import torch

import seq_ref as R

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# The smallest normal fp16 is 2^-14: below it the step is fixed, half of it is 2^-25.  Results of the hardware exponential below
# 2^-126, fp32's smallest normal, become zero: an absolute error of 2^-126 in exp(e A), times the terms it multiplies (states
# and adjoints below 2^10 each, at most 2500 of them added: under 2^-126 2^20 2^12 < 2^-93).
TINY = {torch.float32: 2.0 ** -93, torch.bfloat16: 2.0 ** -93, torch.float16: 2.0 ** -25}


def close(got, want, mag, c, what):
    """|got - want| <= u(t) |want| + c 2^-24 mag (+ what underflow takes)"""
    u = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    g, w = got.detach().double().cpu(), want.double()
    assert tuple(g.shape) == tuple(w.shape), "%s: shape %s, want %s" % (what, tuple(g.shape), tuple(w.shape))
    assert torch.equal(torch.isnan(g), torch.isnan(w)), "%s: NaN in other places" % what
    ok = ~torch.isnan(w)
    slack = u * w.abs() + c * U32 * (1 + u) * mag.double() + TINY[got.dtype]
    bad = ((g - w).abs() > slack) & ok
    if bad.any():
        i = int(((g - w).abs() / slack.clamp(min=1e-300)).nan_to_num(0).argmax())
        raise AssertionError("%s: %d of %d off, worst %.9g want %.9g, allowed %.3g" % (
            what, int(bad.sum()), g.numel(), g.reshape(-1)[i], w.reshape(-1)[i], slack.reshape(-1)[i]))


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ restatements (CPU)
def test_conv_restatement_against_autograd_and_differences():
    g = gen(1)
    x, w, b, st = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((6, 3, 2), (2, 3), (2,), (2, 3, 2)))
    lengths = torch.tensor([6, 1, 0])
    gy, gs = torch.randn(6, 3, 2, generator=g, dtype=torch.float64), torch.randn(2, 3, 2, generator=g, dtype=torch.float64)

    def f(x, w, b, st):
        tot = 0
        for i in range(3):
            full = torch.cat([st[:, i], x[:lengths[i], i]])
            tot = tot + (full[-2:] * gs[:, i]).sum()
            for s in range(int(lengths[i])):
                tot = tot + (torch.nn.functional.silu((full[s:s + 3] * w.t()).sum(0) + b) * gy[s, i]).sum()
        return tot
    assert torch.autograd.gradcheck(f, (x, w, b, st))
    f(x, w, b, st).backward()
    _, _, dx, dw, db, dst = R.conv(x, w, b, True, lengths, st, gy, gs)
    for a, t in ((dx, x), (dw, w), (db, b), (dst, st)):
        assert torch.allclose(a, t.grad, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("gate", [False, True])
def test_scan_restatement_against_autograd_and_differences(gate):
    g = gen(2)
    t, nb, d, n, gr = 4, 2, 4, 3, 2
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)          # noqa: E731
    x, dt, z, B, C, D, bias, st = mk(t, nb, d), mk(t, nb, d), mk(t, nb, d), mk(t, nb, gr, n), mk(t, nb, gr, n), mk(d), mk(d), mk(nb, d, n)
    A = (-torch.rand(d, n, generator=g, dtype=torch.float64)).requires_grad_(True)
    lengths = torch.tensor([4, 2])
    gy, gh = torch.randn(t, nb, d, generator=g, dtype=torch.float64), torch.randn(nb, d, n, generator=g, dtype=torch.float64)

    def f(x, dt, A, B, C, D, z, bias, st):
        tot = 0
        for i in range(nb):
            h = st[i]
            for s in range(int(lengths[i])):
                e = torch.nn.functional.softplus(dt[s, i] + bias)
                of = torch.arange(d) // (d // gr)
                h = torch.exp(e[:, None] * A) * h + (e * x[s, i])[:, None] * B[s, i, of]
                y = (C[s, i, of] * h).sum(-1) + D * x[s, i]
                tot = tot + ((y * torch.nn.functional.silu(z[s, i]) if gate else y) * gy[s, i]).sum()
            tot = tot + (h * gh[i]).sum()
        return tot
    args = (x, dt, A, B, C, D, z, bias, st)
    assert torch.autograd.gradcheck(f, args, check_undefined_grad=False)
    f(*args).backward()
    _, _, gr_ = R.scan(x, dt, A, B, C, D, z if gate else None, bias, True, lengths, st, gy, gh)
    for k, v in (("x", x), ("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("bias", bias), ("state", st)) + ((("z", z),) if gate else ()):
        assert torch.allclose(gr_[k], v.grad, rtol=1e-11, atol=1e-11), k


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_abi_refusals_without_a_gpu():
    from jova_amd import _lib
    p, n8 = ctypes.c_void_p(4096), (ctypes.c_int64 * 12)()
    one, two = (ctypes.c_void_p * 1)(4096), (ctypes.c_void_p * 2)(4096, 4100)
    size, code = (ctypes.c_int64 * 2)(8, 8), (ctypes.c_int32 * 2)(0, 0)
    bad = [
        ("jova_token_embedding_fwd", (p, 7, p, 4, 8, 10, 1.0, p, p, None), "dtype"),
        ("jova_token_embedding_fwd", (None, 0, p, 4, 8, 10, 1.0, p, p, None), "bad argument"),
        ("jova_token_embedding_bwd", (p, 0, p, 2 ** 31, 8, 10, -1, 1.0, p, 0, p, None), "2\\^31"),
        ("jova_token_embedding_bwd", (p, 0, p, 4, 8, 10, -1, 1.0, ctypes.c_void_p(4100), 0, p, None), "16-byte"),
        ("jova_causal_conv_fwd", (p, 8, 8, 0, 4, 2, 8, 9, p, p, 0, 1, None, None, p, None, None), "width 9"),
        ("jova_causal_conv_fwd", (p, 8, 8, 0, 4, 70000, 8, 4, p, p, 0, 1, None, None, p, None, None), "65535"),
        ("jova_causal_conv_bwd", (p, 8, 8, p, 8, 8, 0, 4, 2, 8, 4, p, p, 3, 1, None, None, None, p, p, p, 0, None, p, None), "dtype"),
        ("jova_causal_conv_step", (p, 8, None, p, 0, 2, 8, 4, p, p, 0, 1, p, None), "null pointer"),
        ("jova_selective_scan_fwd", (p, p, p, p, p, p, p, p, 0, 4, 2, 8, 3, 16, n8, 1, None, None, p, None, None, p, None), "bad shape"),
        ("jova_selective_scan_fwd", (p, p, p, p, p, p, p, p, 0, 4, 2, 8, 1, 33, n8, 1, None, None, p, None, None, p, None), "at most 32"),
        ("jova_selective_scan_step", (p, p, p, p, p, p, p, p, 0, 2, 8, 1, 16, n8, 1, None, p, p, None), "null pointer"),
        ("jova_clip_grads", (1, one, one, size, code, 3, 1.0, 1.0, p, p, None), "norm kind"),
        ("jova_clip_grads", (0, one, one, size, code, 2, 1.0, 1.0, p, p, None), "bad argument"),
        ("jova_clip_grads", (1, one, one, size, (ctypes.c_int32 * 1)(5), 2, 1.0, 1.0, p, p, None), "dtype"),
        ("jova_clip_grads", (2, two, two, size, code, 2, 1.0, 1.0, p, p, None), "share memory"),
    ]
    for name, args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            _lib.call(name, *args)


def test_python_refusals_without_a_gpu():
    from jova_amd.nn import functional as F
    from jova_amd.nn.layers import CausalConv1d, Embedding
    from jova_amd.nn.models import ProteinSSM
    from jova_amd.train import clip_grad_norm_
    w, i = torch.randn(10, 4), torch.tensor([1, 2])
    x, cw = torch.randn(5, 2, 4), torch.randn(4, 3)
    A, B = -torch.rand(4, 3), torch.randn(5, 2, 3)
    sc = dict(x=x, dt=x, A=A, B=B, C=B)
    one = dict(x=x[0], dt=x[0], A=A, B=B[0], C=B[0], state=torch.zeros(2, 4, 3))
    G = dict(error=RuntimeError, match="GPU")
    cases = [
        (lambda: F.embedding(i, w), G), (lambda: F.embedding(i.float(), w), dict(error=TypeError)),
        (lambda: F.embedding(i, w.double()), dict(error=TypeError)), (lambda: F.embedding(i, w, padding_idx=10), dict(error=ValueError)),
        (lambda: F.embedding(i, w[0]), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, cw), G), (lambda: F.causal_conv1d(x, torch.randn(4, 9)), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, torch.randn(4, 1)), dict(error=ValueError)), (lambda: F.causal_conv1d(x[0], cw), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, cw, activation="relu"), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, cw, bias=torch.randn(3)), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, cw.bfloat16()), dict(error=TypeError)),
        (lambda: F.causal_conv1d(x, cw, lengths=[5, 5]), dict(error=TypeError)),
        (lambda: F.causal_conv1d(x, cw, lengths=torch.tensor([5])), dict(error=ValueError)),
        (lambda: F.causal_conv1d(x, cw, initial_state=torch.zeros(3, 2, 4)), dict(error=ValueError)),
        (lambda: F.causal_conv1d_step(x[0], torch.zeros(2, 2, 4), cw), G),
        (lambda: F.causal_conv1d_step(x[0], torch.zeros(2, 2, 4), cw.clone().requires_grad_(True)), dict(error=RuntimeError, match="inference")),
        (lambda: F.causal_conv1d_step(x[0], torch.zeros(2, 2, 4).double(), cw), dict(error=TypeError)),
        (lambda: F.selective_scan(**sc), G), (lambda: F.selective_scan(**dict(sc, A=A.half())), dict(error=TypeError)),
        (lambda: F.selective_scan(**dict(sc, A=torch.rand(4, 33))), dict(error=ValueError)),
        (lambda: F.selective_scan(**dict(sc, B=torch.randn(5, 2, 3, 3), C=torch.randn(5, 2, 3, 3))), dict(error=ValueError)),
        (lambda: F.selective_scan(**dict(sc, dt=x[:4])), dict(error=ValueError)),
        (lambda: F.selective_scan(**dict(sc, z=x.half())), dict(error=TypeError)),
        (lambda: F.selective_scan(initial_state=torch.zeros(2, 4, 4), **sc), dict(error=ValueError)),
        (lambda: F.selective_scan_step(**one), G),
        (lambda: F.selective_scan_step(**dict(one, state=torch.zeros(2, 4, 3).transpose(0, 1).contiguous().transpose(0, 1))), dict(error=ValueError)),
        (lambda: F.selective_scan_step(out_state=torch.zeros(2, 4, 4), **one), dict(error=ValueError)),
        (lambda: clip_grad_norm_([w], 1.0), G), (lambda: clip_grad_norm_([w], 1.0, norm_type=3), dict(error=ValueError)),
        (lambda: clip_grad_norm_([w], -1.0), dict(error=ValueError)), (lambda: clip_grad_norm_([w], float("nan")), dict(error=ValueError)),
        (lambda: clip_grad_norm_([w[:, :2]], 1.0), dict(error=ValueError, match="contiguous")),
        (lambda: clip_grad_norm_([w.double()], 1.0), dict(error=TypeError)),
        (lambda: clip_grad_norm_([w], 1.0, out=[w[:5]]), dict(error=ValueError)),
        (lambda: Embedding(5, 4, max_norm=1.0), dict(error=NotImplementedError)), (lambda: Embedding(5, 4, sparse=True), dict(error=NotImplementedError)),
        (lambda: CausalConv1d(4, 9), dict(error=ValueError)), (lambda: ProteinSSM(4, 8, state_dim=33), dict(error=ValueError)),
    ]
    buf = torch.zeros(3, 4, 3)
    cases.append((lambda: F.selective_scan_step(**dict(one, state=buf[:2], out_state=buf[1:])), dict(error=ValueError, match="overlaps")))
    for k, (f, e) in enumerate(cases):
        with pytest.raises(e["error"], match=e.get("match")):
            f()
            raise AssertionError("case %d was not refused" % k)
    assert float(clip_grad_norm_([torch.nn.Parameter(w)], 1.0)) == 0.0                # no gradients: nothing to do


def test_a_grid_too_large_and_a_capture_over_an_eager_graph_are_refused(monkeypatch):
    from jova_amd import _lib
    from jova_amd.nn import functional as F
    p = ctypes.c_void_p(4096)
    with pytest.raises(RuntimeError, match="one grid"):              # 2^29 rows of 8: 2^24 tiles of 256 threads
        _lib.call("jova_token_embedding_bwd", p, 1, p, 2 ** 29, 8, 10, -1, 1.0, p, 0, p, None)

    class Graph:                                                     # stands for the context of a differentiable call
        pass
    now = dict(stream=1, capturing=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now["stream"], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    w, other, x = torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True), torch.ones(2)
    eager = Graph()
    F._note_leaves(eager, x, w, None)
    assert [t is w for t in eager.leaves] == [True]
    now.update(stream=2, capturing=True)
    F._note_leaves(Graph(), x, other)                                # other leaves
    with pytest.raises(RuntimeError, match="eager graph"):
        F._note_leaves(Graph(), x, w)
    now["stream"] = 1
    F._note_leaves(Graph(), x, w)                                    # built on the capture's own stream
    now["stream"] = 2
    del eager
    F._note_leaves(Graph(), x, w)


# ------------------------------------------------------------------------------------------------ embedding (GPU)
EMB = [(1, 1, 1), (3, 5, 7), (64, 10, 22), (2049, 300, 33), (5000, 9049, 22), (300, 70000, 8), (4096, 2, 130), (777, 40, 2056), (0, 6, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,d", EMB)
def test_embedding_and_its_gradient(device, n, vocab, d, dtype):
    """Lookup and gradient by sorted tokens: one token for all, more tokens than rows, rows that are not a vector wide; a third of
    the ids is the padding token.  Rounding: the lookup multiplies once; a token's m rows are m - 1 additions and one product."""
    from jova_amd.nn import functional as F
    g = gen(n + vocab + d)
    w = torch.randn(vocab, d, generator=g).to(dtype)
    idx = torch.randint(vocab, (n,), generator=g)
    pad = vocab - 1 if vocab > 1 else None
    if pad is not None:
        idx[torch.rand(n, generator=g) < 0.33] = pad
    dout = torch.randn(n, d, generator=g).to(dtype)
    scale = 1.7
    want, dw, mag, count = R.embedding(idx, w, dout, scale, pad)
    wd = w.to(device).requires_grad_(True)
    out = F.embedding(idx.to(device), wd, scale=scale, padding_idx=pad)
    close(out, want, want.abs(), 2, "out")
    got, = torch.autograd.grad(out, wd, dout.to(device), retain_graph=True)
    close(got, dw, mag * (count[:, None] + 2), 1, "dweight")
    again, = torch.autograd.grad(out, wd, dout.to(device))
    assert torch.equal(got, again)                                   # the same bits on every call


@pytest.mark.gpu
def test_embedding_gradient_adds_to_an_existing_grad_and_leaves_other_rows(device):
    from jova_amd.nn import functional as F
    g = gen(5)
    w = torch.randn(50, 6, generator=g).to(device).requires_grad_(True)
    before = torch.randn(50, 6, generator=g).to(device)
    w.grad = before.clone()
    idx = torch.tensor([3, 3, 7, 49, 3], device=device, dtype=torch.int32)
    dout = torch.randn(5, 6, generator=g).to(device)
    F.embedding(idx, w, scale=2.0).backward(dout)
    want = before.double().cpu()
    for r, v in enumerate(idx.tolist()):
        want[v] += 2.0 * dout[r].double().cpu()
    close(w.grad, want, want.abs() + 6 * dout.abs().max().cpu(), 6, "grad")
    rest = [v for v in range(50) if v not in (3, 7, 49)]
    assert torch.equal(w.grad[rest], before[rest])


@pytest.mark.gpu
def test_embedding_ids_outside_the_table(device):
    from jova_amd.nn import functional as F
    w = torch.randn(9, 4, device=device, requires_grad=True)
    out = F.embedding(torch.tensor([[0, 9], [-1, 8]], device=device), w)
    assert out.shape == (2, 2, 4) and torch.isnan(out[0, 1]).all() and torch.isnan(out[1, 0]).all() and torch.equal(out[1, 1], w[8])
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert torch.equal(dw.sum(1).cpu(), torch.tensor([4., 0, 0, 0, 0, 0, 0, 0, 4.]))
    with pytest.raises(IndexError):
        F.EmbeddingFunction.raise_if_bad()
    F.EmbeddingFunction.raise_if_bad()                               # (reported once)


@pytest.mark.gpu
def test_embedding_one_hot_token_over_many_tiles(device):
    """90 % of 20000 rows are one token (its run spans hundreds of tiles), next to singles; a strided weight and gradient."""
    from jova_amd.nn import functional as F
    g = gen(11)
    n, v, d = 20000, 1000, 24
    idx = torch.randint(v, (n,), generator=g)
    idx[torch.rand(n, generator=g) < 0.9] = 417
    w = torch.randn(d, v, generator=g).t()
    dout = torch.randn(n, 2 * d, generator=g)[:, ::2]
    want, dw, mag, count = R.embedding(idx, w, dout, 0.5, None)
    wd = w.to(device).requires_grad_(True)
    out = F.embedding(idx.to(device), wd, scale=0.5)
    close(out, want, want.abs(), 2, "out")
    got, = torch.autograd.grad(out, wd, dout.to(device))
    close(got, dw, mag * (count[:, None].sqrt() + 4), 4, "dweight")     # (tile sums added up: far fewer than count roundings in a row)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 600, 300000])
def test_embedding_gradient_of_many_rows(device, vocab):
    """300 001 rows: more than one round per sorting workgroup; one, two and three passes.  The rows are small integers, so every sum is
    exact in fp32 and equals the float64 one."""
    from jova_amd.nn import functional as F
    g = gen(vocab)
    n, d = 300001, 4
    idx = (torch.rand(n, generator=g, dtype=torch.float64) ** 3 * vocab).long()
    idx[::7] = -1                                                    # outside: no gradient
    dout = torch.randint(-4, 5, (n, d), generator=g).float()
    want = torch.zeros(vocab, d, dtype=torch.float64).index_add_(0, idx[idx >= 0], dout[idx >= 0].double())
    w = torch.zeros(vocab, d, device=device, requires_grad=True)
    got, = torch.autograd.grad(F.embedding(idx.to(device), w), w, dout.to(device))
    assert torch.equal(got.double().cpu(), want)
    with pytest.raises(IndexError):
        F.EmbeddingFunction.raise_if_bad()


# ------------------------------------------------------------------------------------------------ convolution (GPU)
CONV = [(1, 1, 1, 2), (3, 2, 5, 4), (70, 3, 33, 3), (64, 2, 256, 4), (131, 1, 260, 8), (200, 4, 24, 5), (5, 7, 64, 6), (129, 2, 10, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,b,d,width", CONV)
def test_conv_forward_backward(device, t, b, d, width, dtype):
    """With a state in front, ragged lengths (0 and 1 among them) and the gradient of the final state.  p: width + 1 roundings of
    the magnitudes, SiLU and its slope a dozen more; dw and dbias add t b terms."""
    from jova_amd.nn import functional as F
    g = gen(t * b + d + width)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype)                                            # noqa: E731
    x, w, bias, st = mk(t, b, d), mk(d, width), mk(d), mk(width - 1, b, d)
    dy, ds = mk(t, b, d), mk(width - 1, b, d)
    lengths = torch.randint(0, t + 1, (b,), generator=g)
    lengths[0] = t
    if b > 2:
        lengths[1], lengths[2] = 0, 1
    for silu in (True, False):
        ref = R.conv(x, w, bias, silu, lengths, st, dy, ds)
        mag = R.conv(x, w, bias, silu, lengths, st, dy, ds, mag=True)
        a = [v.to(device).requires_grad_(True) for v in (x, w, bias, st)]
        y, fin = F.causal_conv1d(a[0], a[1], a[2], "silu" if silu else None, lengths.to(device), a[3], True)
        c = width + 16
        close(y, ref[0], 1.1 * mag[0] + ref[0].abs(), c, "y")
        assert torch.equal(fin.cpu().double(), ref[1])
        got = torch.autograd.grad((y, fin), a, (dy.to(device), ds.to(device)))
        for k, (name, extra) in enumerate((("dx", width), ("dweight", t * b), ("dbias", t * b), ("dstate", width))):
            close(got[k], ref[2 + k], mag[2 + k], c + extra, name)
    y = F.causal_conv1d(x.to(device), w.to(device))                   # no bias, no state, no lengths
    close(y, R.conv(x, w, None, False, None, None)[0], R.conv(x, w, None, False, None, None, mag=True)[0], width + 2, "plain y")


@pytest.mark.gpu
def test_conv_strides_padding_garbage_and_pieces(device):
    """Batch-first and sliced views; NaN behind the ends stays out of every result; a sequence in pieces equals the whole."""
    from jova_amd.nn import functional as F
    g = gen(3)
    t, b, d, width = 37, 3, 20, 4
    wide = torch.randn(b, t, 2 * d, generator=g)
    lengths = torch.tensor([37, 11, 0])
    for i, n in enumerate(lengths.tolist()):
        wide[i, n:] = float("nan")
    w, bias = torch.randn(d, width, generator=g), torch.randn(d, generator=g)
    dy = torch.randn(t, b, d, generator=g)
    dy[12:, 1] = float("inf")
    x = wide.transpose(0, 1)[..., d:]
    clean = torch.nan_to_num(x)
    ref = R.conv(clean, w, bias, True, lengths, None, torch.nan_to_num(dy, posinf=0.0))
    mag = R.conv(clean, w, bias, True, lengths, None, torch.nan_to_num(dy, posinf=0.0), mag=True)
    wd = wide.to(device)
    xd = wd.transpose(0, 1)[..., d:].requires_grad_(True)
    assert not xd.is_contiguous()
    pw, pb = w.to(device).requires_grad_(True), bias.to(device).requires_grad_(True)
    y = F.causal_conv1d(xd, pw, pb, "silu", lengths.to(device))
    got = torch.autograd.grad(y, (xd, pw, pb), dy.to(device))
    close(y, ref[0], 1.1 * mag[0], 20, "y")
    for k, name in enumerate(("dx", "dweight", "dbias")):
        close(got[k], ref[2 + k], mag[2 + k], 20 + t * b, name)
    full = torch.randn(t, b, d, generator=g).to(device)
    whole, end = F.causal_conv1d(full, pw.detach(), pb.detach(), "silu", return_final_state=True)
    st, parts = None, []
    for lo, hi in ((0, 1), (1, 3), (3, 20), (20, 37)):
        p, st = F.causal_conv1d(full[lo:hi], pw.detach(), pb.detach(), "silu", initial_state=st, return_final_state=True)
        parts.append(p)
    assert torch.equal(torch.cat(parts), whole) and torch.equal(st, end)
    st, parts = torch.zeros(width - 1, b, d, device=device), []
    for s in range(t):
        parts.append(F.causal_conv1d_step(full[s], st, pw.detach(), pb.detach(), "silu"))
    assert torch.equal(torch.stack(parts), whole) and torch.equal(st, end)


@pytest.mark.gpu
def test_conv_fp32_weights_on_16_bit_inputs_and_accumulated_gradients(device):
    """Master weights in fp32 next to bf16 activations; a .grad that is there is added to; frozen parameters get none; misaligned rows."""
    from jova_amd.nn import functional as F
    g = gen(8)
    t, b, d, width = 66, 2, 12, 3
    wide = torch.randn(t, b, d + 1, generator=g).bfloat16()
    w, bias, dy = torch.randn(d, width, generator=g), torch.randn(d, generator=g), torch.randn(t, b, d, generator=g).bfloat16()
    x = wide[..., 1:]                                                # two bytes off every vector boundary
    ref = R.conv(x, w, bias, True, None, None, dy)
    mag = R.conv(x, w, bias, True, None, None, dy, mag=True)
    xd = wide.to(device)[..., 1:]
    pw, pb = w.to(device).requires_grad_(True), bias.to(device).requires_grad_(True)
    pw.grad, pb.grad = torch.full_like(pw, 2.0), torch.full_like(pb, -3.0)
    y = F.causal_conv1d(xd, pw, pb, "silu")
    close(y, ref[0], 1.1 * mag[0], 20, "y")
    y.backward(dy.to(device))
    close(pw.grad, ref[3] + 2.0, mag[3] + 2.0, 22 + t * b, "dweight")
    close(pb.grad, ref[4] - 3.0, mag[4] + 3.0, 22 + t * b, "dbias")
    frozen = w.to(device)
    pb.grad = None
    y = F.causal_conv1d(xd, frozen, pb, "silu")
    y.backward(dy.to(device))
    assert frozen.grad is None
    close(pb.grad, ref[4], mag[4], 22 + t * b, "dbias alone")
    lx = xd.clone().requires_grad_(True)
    y = F.causal_conv1d(lx, frozen, None, "silu")
    y.backward(dy.to(device))
    assert lx.grad.dtype == torch.bfloat16 and torch.isfinite(lx.grad).all()
    with pytest.raises(RuntimeError, match="twice differentiable|once_differentiable|does not require grad|once"):
        z = F.causal_conv1d(lx, frozen, None, "silu")
        gx, = torch.autograd.grad(z.float().sum(), lx, create_graph=True)
        gx.float().sum().backward()


# ------------------------------------------------------------------------------------------------ scan (GPU)
def scan_inputs(g, t, b, d, n, gr, dtype):
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype)                                            # noqa: E731
    a = dict(x=mk(t, b, d), dt=mk(t, b, d), A=-torch.rand(d, n, generator=g) * 4 - 0.01, B=mk(t, b, gr, n), C=mk(t, b, gr, n),
             D=torch.randn(d, generator=g), z=mk(t, b, d), bias=torch.randn(d, generator=g) - 2.0,
             state=torch.randn(b, d, n, generator=g))
    return a, mk(t, b, d), torch.randn(b, d, n, generator=g)


# y: per step the exponent (softplus, two products, exp), the state's product and sum: under 16 roundings of magnitudes that decay
# afterwards; the n states and the gate add n + 16.  The gradients run the same recurrence twice (states, adjoint): twice that.
def scan_c(t, n):
    return 16 * t + n + 32


SCAN = [(1, 1, 1, 1, 1), (2, 3, 5, 3, 1), (16, 2, 64, 16, 1), (17, 2, 66, 16, 2), (33, 1, 20, 8, 1), (70, 3, 130, 11, 1), (19, 2, 12, 32, 3),
        (150, 1, 64, 4, 1), (40, 2, 100, 16, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,b,d,n,gr", SCAN)
def test_scan_forward_backward(device, t, b, d, n, gr, dtype):
    from jova_amd.nn import functional as F
    g = gen(t + b + d + n)
    a, dy, dh = scan_inputs(g, t, b, d, n, gr, dtype)
    lengths = torch.randint(0, t + 1, (b,), generator=g)
    lengths[0] = t
    if b > 2:
        lengths[1], lengths[2] = 0, 1
    keys = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")
    y0, h0, gr0 = R.scan(*(a[k] for k in keys[:8]), True, lengths, a["state"], dy, dh)
    ym, hm, grm = R.scan(*(a[k] for k in keys[:8]), True, lengths, a["state"], dy, dh, mag=True)
    v = {k: a[k].to(device).requires_grad_(True) for k in keys}
    y, h = F.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, lengths.to(device), v["state"], True)
    c = scan_c(t, n)
    close(y, y0, ym, c, "y")
    close(h, h0, hm, c, "state")
    got = torch.autograd.grad((y, h), [v[k] for k in keys], (dy.to(device), dh.to(device)), retain_graph=True)
    for k, x in zip(keys, got):
        extra = {"A": t * b, "D": t * b, "bias": t * b, "B": d // gr, "C": d // gr}.get(k, 0)
        close(x, gr0[k], grm[k], 2 * c + extra, "d" + k)
    again = torch.autograd.grad((y, h), [v[k] for k in keys], (dy.to(device), dh.to(device)))
    assert all(torch.equal(p, q) for p, q in zip(got, again))        # no atomics


@pytest.mark.gpu
@pytest.mark.parametrize("softplus", [False, True])
def test_scan_optional_arguments(device, softplus):
    """Without D, z, bias, state, lengths; B and C without a group axis; only the outputs' gradient, only the state's."""
    from jova_amd.nn import functional as F
    g = gen(9)
    t, b, d, n = 21, 2, 24, 16
    a, dy, dh = scan_inputs(g, t, b, d, n, 1, torch.float32)
    if not softplus:
        a["dt"] = a["dt"].abs() * 0.1
    want = {}
    for which in ("y", "h"):
        args = [a[k] for k in ("x", "dt", "A", "B", "C")] + [None, None, None, softplus, None, None]
        gy, gh = (dy, None) if which == "y" else (None, dh)
        want[which] = R.scan(*args, gy, gh), R.scan(*args, gy, gh, mag=True)
    v = {k: a[k].to(device).requires_grad_(True) for k in ("x", "dt", "A", "B", "C")}
    y, h = F.selective_scan(v["x"], v["dt"], v["A"], v["B"].squeeze(2), v["C"].squeeze(2), dt_softplus=softplus, return_final_state=True)
    for which, out, go in (("y", y, dy), ("h", h, dh)):
        ref, mag = want[which]
        close(out, ref[0 if which == "y" else 1], mag[0 if which == "y" else 1], scan_c(t, n), which)
        got = torch.autograd.grad(out, list(v.values()), go.to(device), retain_graph=True, allow_unused=True)
        for k, x in zip(v, got):
            close(x, ref[2][k], mag[2][k], 2 * scan_c(t, n) + t * b + d, "d%s from %s" % (k, which))


@pytest.mark.gpu
def test_scan_strides_garbage_pieces_and_single_steps(device):
    """Views of one projection (channels sliced, batch first), NaN and infinities behind the ends, the sequence in pieces and
    one step at a time."""
    from jova_amd.nn import functional as F
    g = gen(21)
    t, b, d, n, gr = 45, 3, 40, 16, 2
    lengths = torch.tensor([45, 17, 0])
    width = 3 * d + 2 * gr * n
    big = torch.randn(b, t, width, generator=g)
    A, D, bias = -torch.rand(d, n, generator=g) - 0.05, torch.randn(d, generator=g), torch.randn(d, generator=g) - 2
    dy = torch.randn(t, b, d, generator=g)

    def cut(p):
        p = p.transpose(0, 1)
        return dict(x=p[..., :d], dt=p[..., d:2 * d], z=p[..., 2 * d:3 * d], B=p[..., 3 * d:3 * d + gr * n].unflatten(-1, (gr, n)),
                    C=p[..., 3 * d + gr * n:].unflatten(-1, (gr, n)))
    clean = cut(big)
    order = lambda s, a, d_, bi: (s["x"], s["dt"], a, s["B"], s["C"], d_, s["z"], bi)                 # noqa: E731
    ref = R.scan(*order(clean, A, D, bias), True, lengths, None, dy)
    mag = R.scan(*order(clean, A, D, bias), True, lengths, None, dy, mag=True)
    dirty = big.clone()
    for i, m in enumerate(lengths.tolist()):
        dirty[i, m:, ::2], dirty[i, m:, 1::2] = float("nan"), float("inf")
    dyd = dy.clone()
    for i, m in enumerate(lengths.tolist()):
        dyd[m:, i] = float("nan")
    leaf = dirty.to(device).requires_grad_(True)
    s = cut(leaf)
    Ad, Dd, bd = (p.to(device).requires_grad_(True) for p in (A, D, bias))
    y, h = F.selective_scan(*order(s, Ad, Dd, bd), True, lengths.to(device), None, True)
    close(y, ref[0], mag[0], scan_c(t, n), "y")
    close(h, ref[1], mag[1], scan_c(t, n), "state")
    gl, gA, gD, gb = torch.autograd.grad(y, (leaf, Ad, Dd, bd), dyd.to(device))
    for k, x in cut(gl).items():
        close(x, ref[2][k], mag[2][k], 2 * scan_c(t, n) + d, "d" + k)
    for k, x in (("A", gA), ("D", gD), ("bias", gb)):
        close(x, ref[2][k], mag[2][k], 2 * scan_c(t, n) + t * b, "d" + k)
    # in pieces, and one step at a time (the same arithmetic per step; the pieces may be cut differently inside)
    c = cut(big.to(device))
    args = (Ad.detach(), Dd.detach(), bd.detach())
    whole, end = F.selective_scan(*order(c, *args), True, return_final_state=True)
    wmag = R.scan(*order(clean, A, D, bias), True, None, None, mag=True)
    st, parts = None, []
    for lo, hi in ((0, 1), (1, 18), (18, 45)):
        p, st = F.selective_scan(*order({k: v[lo:hi] for k, v in c.items()}, *args), True, initial_state=st, return_final_state=True)
        parts.append(p)
    close(torch.cat(parts), whole.double().cpu(), wmag[0], 2 * scan_c(t, n), "pieces")
    close(st, end.double().cpu(), wmag[1], 2 * scan_c(t, n), "pieces' state")
    st, parts = torch.zeros(b, d, n, device=device), []
    for i in range(t):
        o = {k: v[i] for k, v in c.items()}
        parts.append(F.selective_scan_step(o["x"], o["dt"], args[0], o["B"], o["C"], st, args[1], o["z"], args[2], True))
    close(torch.stack(parts), whole.double().cpu(), wmag[0], 2 * scan_c(t, n), "steps")
    close(st, end.double().cpu(), wmag[1], 2 * scan_c(t, n), "steps' state")


@pytest.mark.gpu
def test_scan_long_sequence_and_extreme_time_steps(device):
    """2500 steps of one sequence (the time axis is split there); time steps from 1e-7 to 40, where exp(e A) runs from 1 to 0."""
    from jova_amd.nn import functional as F
    g = gen(31)
    t, b, d, n = 2500, 1, 18, 16
    a, dy, dh = scan_inputs(g, t, b, d, n, 1, torch.float32)
    a["dt"] = torch.linspace(-16, 40, d).expand(t, b, d) + 0.1 * a["dt"]
    keys = ("x", "dt", "A", "B", "C", "D", "z")
    ref = R.scan(*(a[k] for k in keys), None, True, None, a["state"], dy, dh)
    mag = R.scan(*(a[k] for k in keys), None, True, None, a["state"], dy, dh, mag=True)
    v = {k: a[k].to(device).requires_grad_(True) for k in keys + ("state",)}
    y, h = F.selective_scan(*(v[k] for k in keys), None, True, None, v["state"], True)
    # (the worst path of 2500 steps, 16 roundings each, is not met: a quarter of it holds with the errors' signs mixed)
    c = scan_c(t, n) / 4
    close(y, ref[0], mag[0], c, "y")
    close(h, ref[1], mag[1], c, "state")
    got = torch.autograd.grad((y, h), list(v.values()), (dy.to(device), dh.to(device)))
    for k, x in zip(v, got):
        close(x, ref[2][k], mag[2][k], 2 * c, "d" + k)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,n", [(3, 16), (3, 20), (300, 4)])
def test_scan_ragged_batches_over_several_chunks(device, batch, n):
    """Sequences that end in different chunks of the split time axis (and more of them than a workgroup ranks): against runs of
    each sequence by itself, cut to its length, whose time axis is split elsewhere or not at all."""
    from jova_amd.nn import functional as F
    g = gen(batch + n)
    t, d = (700, 24) if batch == 3 else (40, 24)
    a, dy, dh = scan_inputs(g, t, batch, d, n, 1, torch.float32)
    lengths = torch.randint(0, t + 1, (batch,), generator=g)
    lengths[:3] = torch.tensor([t, t // 5, 0])
    keys = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")

    def run(v, dy, dh, lens):
        v = {k: x.to(device).requires_grad_(True) for k, x in v.items()}
        y, h = F.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, lens, v["state"], True)
        gr = torch.autograd.grad((y, h), [v[k] for k in keys], (dy.to(device), dh.to(device)))
        return y.detach(), h.detach(), dict(zip(keys, gr))
    y, h, gr = run(a, dy, dh, lengths.to(device))
    mag = R.scan(*(a[k] for k in keys[:8]), True, lengths, a["state"], dy, dh, mag=True) if batch == 3 else None
    c = 4 * scan_c(t, n)
    tot = {k: torch.zeros(a[k].shape, dtype=torch.float64) for k in ("A", "D", "bias")}
    for i in (range(batch) if batch == 3 else (0, 1, 2, 150, 299)):
        m = int(lengths[i])
        one = {k: (x[:m, i:i + 1] if x.dim() >= 3 and k != "state" else x[i:i + 1] if k == "state" else x) for k, x in a.items()}
        y1, h1, g1 = run(one, dy[:m, i:i + 1], dh[i:i + 1], None)
        mi = R.scan(*(one[k] for k in keys[:8]), True, None, one["state"], dy[:m, i:i + 1], dh[i:i + 1], mag=True) if m else None
        if m:
            close(y[:m, i:i + 1], y1.double().cpu(), mi[0], c, "y")
            for k in ("x", "dt", "z", "B", "C"):
                close(gr[k][:m, i:i + 1], g1[k].double().cpu(), mi[2][k], 2 * c, "d" + k)
            close(h[i:i + 1], h1.double().cpu(), mi[1], c, "state")
            close(gr["state"][i:i + 1], g1["state"].double().cpu(), mi[2]["state"], 2 * c, "dstate")
        else:
            assert torch.equal(h[i], a["state"][i].to(device)) and torch.equal(gr["state"][i], dh[i].to(device))
        assert float(y[m:, i].abs().sum()) == 0.0 and all(float(gr[k][m:, i].abs().sum()) == 0.0 for k in ("x", "dt", "z", "B", "C"))
        for k in tot:
            tot[k] += g1[k].double().cpu()
    if batch == 3:
        for k in tot:
            close(gr[k], tot[k], mag[2][k], 2 * c + t * batch, "d" + k)


@pytest.mark.gpu
def test_scan_growing_states_and_silent_channels(device):
    """A > 0 over a split time axis: a channel without input stays at zero although its factor over a chunk overflows."""
    from jova_amd.nn import functional as F
    t, d = 1200, 4
    x = torch.zeros(t, 1, d, device=device)
    x[:, :, 0] = 1e-3
    dt = torch.full((t, 1, d), 0.5, device=device)
    A = torch.full((d, 2), 0.9, device=device)
    A[0] = -1.0
    B = torch.ones(t, 1, 2, device=device)
    y, h = F.selective_scan(x, dt, A, B, B, return_final_state=True)
    assert float(y[..., 1:].abs().max()) == 0.0 and float(h[:, 1:].abs().max()) == 0.0
    end = 0.5e-3 / (1 - math.exp(-0.5))                              # the geometric series' limit
    assert abs(float(h[0, 0, 0]) - end) <= 1e-5 * end


@pytest.mark.gpu
def test_scan_and_conv_gradients_against_differences(device):
    """The directional derivative of the fp32 forward pass, by a central difference of step s: its truncation error is s^2 / 6 times
    the third derivative (O(1) here) and its rounding error 2^-24 |f| / s, so 1e-3 of the gradient's scale at s = 1e-2."""
    from jova_amd.nn import functional as F
    g = gen(41)
    t, b, d, n = 12, 2, 8, 4
    a, dy, _ = scan_inputs(g, t, b, d, n, 1, torch.float32)
    keys = ("x", "dt", "A", "B", "C", "D", "z", "bias")
    v = {k: a[k].to(device) for k in keys}
    cw, cb = torch.randn(d, 4, generator=g).to(device), torch.randn(d, generator=g).to(device)
    gy = dy.to(device)

    def f(v, cw):
        u = F.causal_conv1d(v["x"], cw, cb, "silu")
        y = F.selective_scan(u, v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True)
        return (y.double() * gy.double()).sum()
    leaves = {k: x.clone().requires_grad_(True) for k, x in v.items()}
    lw = cw.clone().requires_grad_(True)
    grads = torch.autograd.grad(f(leaves, lw), list(leaves.values()) + [lw])
    s = 1e-2
    for k, gr in zip(list(keys) + ["conv"], grads):
        e = torch.randn(gr.shape, generator=g).to(device)
        e /= e.norm()
        if k == "conv":
            diff = (f(v, cw + s * e) - f(v, cw - s * e)) / (2 * s)
        else:
            diff = (f({**v, k: v[k] + s * e}, cw) - f({**v, k: v[k] - s * e}, cw)) / (2 * s)
        along = float((gr.double() * e.double()).sum())
        assert abs(float(diff) - along) <= 1e-3 * max(1.0, float(gr.norm())), (k, float(diff), along)


# ------------------------------------------------------------------------------------------------ clipping (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("kind", [2.0, 1.0, float("inf")])
@pytest.mark.parametrize("sizes", [[1], [5, 0, 4097], [64] * 130, [100000, 3, 17, 8192]])
def test_clip_norm_and_scaling(device, sizes, kind):
    """In place, into outputs and below the bound; types mixed; more tensors than one call takes.  The norm is summed in fp64 and
    rounded twice, the coefficient takes three roundings, the product one."""
    from jova_amd.train import clip_grad_norm_
    g = gen(len(sizes))
    dts = [DTYPES[i % 3] for i in range(len(sizes))]
    grads = [torch.randn(n, generator=g).to(t) for n, t in zip(sizes, dts)]
    flat = torch.cat([x.double() for x in grads])
    norm = float(flat.abs().max() if kind == float("inf") else flat.norm(p=kind))
    for max_norm in (norm * 0.3, norm * 2):
        c = min(1.0, max_norm / (norm + 1e-6))
        dev = [x.to(device) for x in grads]
        keep = [x.clone() for x in dev]
        out = [torch.full_like(x, 7.0) for x in dev]
        got = clip_grad_norm_(dev, max_norm, norm_type=kind, out=out)
        assert got.shape == () and abs(float(got) - norm) <= 4 * U32 * norm
        for x, o, k, r in zip(dev, out, keep, grads):
            assert torch.equal(x, k)
            close(o, r.double() * c, r.double().abs() * c, 8, "out")
        params = [torch.nn.Parameter(torch.zeros_like(x)) for x in dev] + [torch.nn.Parameter(torch.zeros(3, device=device))]
        for p, x in zip(params, dev):
            p.grad = x
        assert float(clip_grad_norm_(params, max_norm, norm_type=kind)) == float(got)
        assert all(torch.equal(p.grad, o) for p, o in zip(params, out))


@pytest.mark.gpu
def test_clip_extremes(device):
    from jova_amd.train import clip_grad_norm_
    w = torch.ones(100, device=device)
    for lists in (([w, w], None), ([w[:60], w[40:]], None), ([w[:50]], [w[10:60]])):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grad_norm_(lists[0], 1.0, out=lists[1])
    odd = torch.arange(40000, device=device, dtype=torch.float32)[1:].sub_(20000.0)           # not on a 16-byte boundary
    want = odd.double().norm()
    clip_grad_norm_([odd], 1.0)
    assert abs(float(odd.double().norm()) - 1.0) <= 1e-6 and float(want) > 1e6
    big = torch.full((1000,), 3e38, device=device)
    keep = big.clone()
    n = clip_grad_norm_([big[:1]], 1.0)
    assert abs(float(n) - 3e38) < 1e33 and float(big[0]) == pytest.approx(1.0, rel=1e-6)
    big.copy_(keep)
    n = clip_grad_norm_([big], 1.0)                                  # 3e38 sqrt(1000) is no fp32: inf, and the gradients become 0, as in torch
    ref = keep.cpu().clone().requires_grad_(True)
    ref.grad = keep.cpu().clone()
    torch.nn.utils.clip_grad_norm_([ref], 1.0)
    assert math.isinf(float(n)) and torch.equal(big.cpu(), ref.grad)
    for bad in (float("nan"), float("inf")):
        for kind in (2.0, float("inf"), 1.0):
            x = torch.ones(5000, device=device)
            x[4321] = bad
            ref = torch.zeros(5000, requires_grad=True)
            ref.grad = x.cpu().clone()
            want = torch.nn.utils.clip_grad_norm_([ref], 1.0, norm_type=kind)
            got = clip_grad_norm_([x], 1.0, norm_type=kind)
            assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)) and torch.equal(torch.isinf(got.cpu()), torch.isinf(want))
            assert torch.equal(torch.nan_to_num(x.cpu(), nan=-1.0), torch.nan_to_num(ref.grad, nan=-1.0))
    assert float(clip_grad_norm_([torch.empty(0, device=device)], 1.0)) == 0.0


# ------------------------------------------------------------------------------------------------ together
def _net(device, seed=4):
    from jova_amd.nn.models import ProteinSSM, ProteinWords
    torch.manual_seed(seed)
    rng = __import__("numpy").random.RandomState(seed)
    prof = {"P%d" % i: rng.randint(0, 30, size=(n, 3)) for i, n in enumerate((9, 1, 23))}
    words = ProteinWords(prof, 30, 5).to(device)
    ssm = ProteinSSM(15, 24, state_dim=8).to(device)
    return prof, words, ssm


@pytest.mark.gpu
def test_words_to_scan_encoder_against_its_restatement(device):
    """ProteinWords -> ProteinSSM (embedding, convolution, scan and the linear products in one run) against float64; the padded rows
    change nothing; single segments through ``step`` equal the whole sequence."""
    prof, words, ssm = _net(device)
    x, ln = words([("s", "P0"), ("s", "P1"), ("s", "P2")])
    assert x.shape == (23, 3, 15) and ln.tolist() == [9, 1, 23]
    out = ssm((x, ln))
    p = {k: v.detach().double().cpu() for k, v in ssm.named_parameters()}
    w = words.embedding.weight.detach().double().cpu()
    xs = torch.zeros(23, 3, 15, dtype=torch.float64)
    for i, k in enumerate(prof):
        xs[:prof[k].shape[0], i] = (w[torch.from_numpy(prof[k])] * 5 ** 0.5).reshape(-1, 15)
    assert float((x.detach().double().cpu() - xs).abs().max()) <= 2 * U32 * float(xs.abs().max())
    h = xs @ p["in_proj.weight"].t()
    u = R.conv(h[..., :48], p["conv.weight"], p["conv.bias"], True, ln.cpu(), None)[0]
    q = u @ p["x_proj.weight"].t()
    r, n = ssm.dt_rank, 8
    y = R.scan(u, q[..., :r] @ p["dt_proj.weight"].t(), -torch.exp(p["A_log"]), q[..., r:r + n].unsqueeze(2), q[..., r + n:].unsqueeze(2),
               p["D"], h[..., 48:], p["dt_bias"], True, ln.cpu(), None)[0]
    want = torch.relu(y @ p["out_proj.weight"].t() + p["out_proj.bias"])
    # five products of at most 48 terms, a convolution and 23 steps of the scan in a row: under 1000 roundings of the largest value
    assert float((out.detach().double().cpu() - want).abs().max()) <= 1000 * U32 * float(want.abs().max())
    st, got = ssm.new_state(1, device), []
    for s in range(23):
        got.append(ssm.step(x[s, 2:3].detach(), st))
    assert float((torch.stack(got)[:, 0].double().cpu() - want[:, 2]).abs().max()) <= 1000 * U32 * float(want.abs().max())
    out.square().sum().backward()
    for k, v in list(words.named_parameters()) + list(ssm.named_parameters()):
        assert v.grad is not None and torch.isfinite(v.grad).all() and float(v.grad.abs().max()) > 0, k
    assert float(words.embedding.weight.grad[30].abs().max()) == 0.0                  # the padding word


@pytest.mark.gpu
def test_ssm_view_trains_with_clipping_in_the_joint_model(device):
    """The "ssm" protein view through create_integrated_net and Trainer with max_grad_norm: the norm that the trainer reports is the
    gradients', and the update is that of the clipped gradients."""
    from test_gpu_ops import _e2e_setup
    import helpers as H
    from jova_amd.train import Trainer, create_integrated_net
    z, hp, hparams, net0, batch = _e2e_setup(device)
    hparams = dict(hparams, optimizer="sgd", optimizer__global__lr=0.1, optimizer__global__weight_decay=0.0, max_grad_norm=0.05)
    hparams["prot"] = dict(hparams["prot"], model_types=["ssm"], ssm_hidden_dim=20)
    torch.manual_seed(3)
    net = create_integrated_net(hparams, H.profile(z)).to(device).train()
    tr = Trainer(net, hparams)
    tr.flat.zero_grad()
    loss, _ = tr.forward_loss(batch)
    loss.backward()
    g, before = tr.flat.grad.clone(), tr.flat.data.clone()
    norm = float(g.double().norm())
    assert norm > 0.05
    tr.step(batch)
    # (the second backward repeats the first up to the order of the other layers' atomics)
    assert abs(float(tr.grad_norm) - norm) <= 1e-3 * norm
    moved = (before - tr.flat.data).double() / 0.1
    assert abs(float(moved.norm()) - 0.05) <= 1e-3 * 0.05 + 2 * U32 * float(before.double().norm()) / 0.1
    assert float((moved - g.double() * (0.05 / norm)).norm()) <= 2e-3 * 0.05 + 2 * U32 * float(before.double().norm()) / 0.1


@pytest.mark.gpu
def test_forward_backward_and_clip_in_a_captured_graph(device):
    """Embedding -> convolution -> scan, their gradients and the clipping captured into two graphs, replayed in turn with eager work
    and synchronisation between, against the eager results bit for bit."""
    from jova_amd.nn import functional as F
    from jova_amd.train import clip_grad_norm_
    g = gen(51)
    t, b, d, v, n = 70, 2, 32, 40, 16

    def build(seed):
        g = gen(seed)
        idx = torch.randint(v, (t, b), generator=g).to(device)
        fixed = dict(dt=torch.randn(t, b, d, generator=g).to(device), B=torch.randn(t, b, n, generator=g).to(device),
                     C=torch.randn(t, b, n, generator=g).to(device), gy=torch.randn(t, b, d, generator=g).to(device))
        start = [torch.randn(v, d, generator=g), torch.randn(d, 4, generator=g), torch.randn(d, generator=g), -torch.rand(d, n, generator=g) - .1]

        def leaves():
            return [p.to(device).requires_grad_(True) for p in start]

        def run(w):
            x = F.embedding(idx, w[0], scale=2.0, padding_idx=0)
            u = F.causal_conv1d(x, w[1], w[2], "silu")
            y = F.selective_scan(u, fixed["dt"], w[3], fixed["B"], fixed["C"], dt_softplus=True)
            gr = torch.autograd.grad(y, w, fixed["gy"])
            out = [torch.empty_like(k) for k in gr]
            return [y.detach(), clip_grad_norm_(list(gr), 1.0, out=out)] + out
        return idx, fixed, leaves, run
    made = []
    for seed in (1, 2):
        idx, fixed, leaves, run = build(seed)
        w = leaves()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(w)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(w)
        made.append((idx, fixed, leaves, run, w, graph, outs))
    for trial in range(4):
        for idx, fixed, leaves, run, w, graph, outs in made:
            fixed["gy"].mul_(1.0 + trial)
            idx.copy_(torch.randint(v, (t, b), generator=g))
        for _, _, _, _, _, graph, _ in made:
            graph.replay()
        torch.cuda.synchronize()
        for idx, fixed, leaves, run, w, graph, outs in made:
            got = [o.clone() for o in outs]
            eager = run(leaves())
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, eager)), trial


@pytest.mark.gpu
def test_other_stream_and_empty_shapes(device):
    from jova_amd.nn import functional as F
    g = gen(61)
    x, w = torch.randn(30, 2, 16, generator=g).to(device), torch.randn(16, 4, generator=g).to(device)
    A, B = -torch.rand(16, 8, generator=g).to(device), torch.randn(30, 2, 8, generator=g).to(device)
    want = F.selective_scan(F.causal_conv1d(x, w), x, A, B, B, dt_softplus=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.selective_scan(F.causal_conv1d(x, w), x, A, B, B, dt_softplus=True)
    s.synchronize()
    assert torch.equal(got, want)
    for shape in ((0, 2, 16), (30, 0, 16), (0, 0, 16)):
        e = torch.empty(shape, device=device).requires_grad_(True)
        wl = w.clone().requires_grad_(True)
        y, st = F.causal_conv1d(e, wl, return_final_state=True)
        assert y.shape == shape and st.shape == (3, shape[1], 16) and float(st.abs().sum()) == 0.0
        ge, gw = torch.autograd.grad(y.sum() + st.sum(), (e, wl))
        assert ge.shape == shape and float(gw.abs().max()) == 0.0
        Bl, Al = torch.empty(shape[:2] + (8,), device=device).requires_grad_(True), A.clone().requires_grad_(True)
        h0 = torch.randn(shape[1], 16, 8, device=device).requires_grad_(True)
        y, h = F.selective_scan(e, e, Al, Bl, Bl, initial_state=h0, return_final_state=True)
        assert y.shape == shape and torch.equal(h, h0)
        gh, gA = torch.autograd.grad(h.sum() + y.sum(), (h0, Al))
        assert torch.equal(gh, torch.ones_like(h0)) and float(gA.abs().max()) == 0.0


@pytest.mark.gpu
def test_scan_gradients_behind_the_end_of_an_overflowed_sequence(device):
    """A state that has grown to infinity: its own gradients are not finite, the rows behind its end and the other sequence are."""
    from jova_amd.nn import functional as F
    t, d, n = 21, 4, 2
    ones = torch.ones(t, 2, d, device=device)
    x, dt = ones.clone(), ones * torch.tensor([40.0, 0.1], device=device)[:, None]
    B = torch.ones(t, 2, n, device=device)
    leaves = [v.clone().requires_grad_(True) for v in (x, dt, B, B)]
    A = torch.ones(d, n, device=device)
    y = F.selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3], lengths=torch.tensor([11, 13], device=device))
    assert not bool(torch.isfinite(y[10, 0]).any()) and float(y[11:, 0].abs().max()) == 0.0
    for g in torch.autograd.grad(y, leaves, torch.ones_like(y)):
        assert float(g[11:, 0].abs().max()) == 0.0 and float(g[13:, 1].abs().max()) == 0.0
        assert bool(torch.isfinite(g[:, 1]).all())


@pytest.mark.gpu
def test_a_state_moved_on_in_place_is_noticed_by_the_graph_that_saved_it(device):
    from jova_amd.nn import functional as F
    x, state = torch.randn(5, 2, 8, device=device), torch.randn(3, 2, 8, device=device)
    w = torch.randn(8, 4, device=device, requires_grad=True)
    y = F.causal_conv1d(x, w, initial_state=state)
    with torch.no_grad():
        F.causal_conv1d_step(x[0], state, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h, version = torch.zeros(2, 8, 4, device=device), 0
    with torch.no_grad():
        B = torch.randn(2, 4, device=device)
        for _ in range(2):
            F.selective_scan_step(x[0], x[0], -torch.ones(8, 4, device=device), B, B, h)
            assert h._version > version
            version = h._version
    with torch.inference_mode():
        state = torch.zeros(3, 2, 8, device=device)
        F.causal_conv1d_step(x[0], state, w)
        assert torch.equal(state[2], x[0])


@pytest.mark.gpu
def test_scan_backward_whose_chunks_are_cut_into_pieces(device):
    """So many sequences that the time axis is cut into two chunks only, and the adjoint pass over the second into pieces."""
    from jova_amd.nn import functional as F
    g, t, b, d, n = gen(81), 620, 300, 2, 3
    a, dy, dh = scan_inputs(g, t, b, d, n, 1, torch.float32)
    lengths = torch.randint(0, t + 1, (b,), generator=g)
    lengths[:4] = torch.tensor([t, t - 1, 330, 0])
    keys = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")
    v = {k: x.to(device).requires_grad_(True) for k, x in a.items()}
    y, h = F.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, lengths.to(device), v["state"], True)
    got = dict(zip(keys, torch.autograd.grad((y, h), [v[k] for k in keys], (dy.to(device), dh.to(device)))))
    want, mag = (R.scan(*(a[k] for k in keys[:8]), True, lengths, a["state"], dy, dh, mag=m) for m in (False, True))
    c = scan_c(t, n)
    close(y, want[0], mag[0], c, "y")
    close(h, want[1], mag[1], c, "state")
    for k in keys:                                                   # (the parameters' sums run over the batch too)
        close(got[k], want[2][k], mag[2][k], 2 * c + (t * b if k in ("A", "D", "bias") else 0), "d" + k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d,width", [(1, 1, 2), (3, 16, 4), (2, 33, 8), (2, 600, 3)])
def test_conv_over_no_steps_hands_the_state_and_its_gradient_through(device, b, d, width, dtype):
    """A piece of zero steps: the state that is returned is the one that came in, and so is its gradient (zeros without one)."""
    from jova_amd.nn import functional as F
    g = gen(b + d + width)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)                                 # noqa: E731
    x, w, bias, st, ds = mk(5, b, d), mk(d, width), mk(d), mk(width - 1, b, d).requires_grad_(True), mk(width - 1, b, d)
    pw, pb = w.clone().requires_grad_(True), bias.clone().requires_grad_(True)

    def poison():                                                    # the memory that the next allocation of this size gets
        torch.full_like(st, float("nan"))
    for lengths in (None, torch.zeros(b, dtype=torch.int32, device=device)):
        y, fin = F.causal_conv1d(x[:0], pw, pb, "silu", lengths, st, True)
        assert y.shape == (0, b, d) and torch.equal(fin, st)
        poison()
        got = torch.autograd.grad(fin, (st, pw, pb), ds, retain_graph=True)
        assert torch.equal(got[0], ds) and float(got[1].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0
        poison()
        got, = torch.autograd.grad(y, st, torch.empty_like(y))
        assert float(got.abs().max()) == 0.0
    got = []
    for cuts in ((0, 3, 5), (0, 0, 3, 3, 5, 5)):                     # pieces of no steps between the others change nothing
        s = st
        for lo, hi in zip(cuts, cuts[1:]):
            y, s = F.causal_conv1d(x[lo:hi], w, bias, "silu", initial_state=s, return_final_state=True)
            poison()
        got.append(torch.autograd.grad(s, st, ds)[0])
    assert torch.equal(got[0], got[1])


@pytest.mark.gpu
def test_gradients_that_nobody_asked_for_leave_an_existing_grad_alone(device):
    """torch.autograd.grad next to a .grad that is there: what was asked for is returned, .grad stays as it is, hooks see what
    backward() adds."""
    from jova_amd.nn import functional as F
    g = gen(91)
    x, w, b = (torch.randn(*s, generator=g).to(device).requires_grad_(True) for s in ((20, 2, 12), (12, 4), (12,)))
    table, idx, dout = torch.randn(9, 12, generator=g).to(device).requires_grad_(True), torch.randint(9, (20, 2), generator=g).to(device), x.detach()
    calls = {"conv": (lambda: F.causal_conv1d(x, w, b, "silu"), (w, b)), "embedding": (lambda: F.embedding(idx, table), (table,)),
             "both": (lambda: F.causal_conv1d(F.embedding(idx, table), w, b, "silu"), (table, w, b))}
    for name, (call, params) in calls.items():
        for p in params:
            p.grad = None
        want = torch.autograd.grad(call(), params, dout)
        for p in params:
            p.grad = torch.full_like(p, 3.0)
        if name == "conv":
            torch.autograd.grad(call(), x, dout)
            assert all(float((p.grad - 3.0).abs().max()) == 0.0 for p in params), name
        got = torch.autograd.grad(call(), params, dout)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), name
        assert all(float((p.grad - 3.0).abs().max()) == 0.0 for p in params), name
        seen, hooks = [], [p.register_hook(lambda v: seen.append(v)) for p in params]
        at = [p.grad.data_ptr() for p in params]
        call().backward(dout)
        for h in hooks:
            h.remove()
        assert len(seen) == len(params) and all(torch.is_tensor(v) for v in seen), name
        assert all(torch.equal(p.grad, q + 3.0) and p.grad.data_ptr() == a for p, q, a in zip(params, want, at)), name


@pytest.mark.gpu
def test_gradients_of_a_flat_buffer_are_added_in_place(device):
    """The trainer's own gradients (views of FlatParameters' buffer): added to by the kernels, through hooks where there are some."""
    from jova_amd.nn.layers import CausalConv1d, Embedding
    from jova_amd.train import FlatParameters
    torch.manual_seed(7)
    net = torch.nn.Sequential(Embedding(11, 10, padding_idx=3, scale=2.0), CausalConv1d(10, 3)).to(device)
    idx = torch.randint(11, (40, 2), generator=gen(92)).to(device)
    params = list(net.parameters())
    want = torch.autograd.grad(net(idx).square().sum(), params)
    flat = FlatParameters(net)
    flat.grad.fill_(0.5)
    for trial in range(2):
        seen = []
        hooks = [p.register_hook(lambda v: seen.append(v)) for p in params] if trial else []
        net(idx).square().sum().backward()
        assert len(seen) == len(hooks) and all(torch.is_tensor(v) for v in seen)
        for p, q in zip(params, want):
            assert p.grad.untyped_storage().data_ptr() == flat.grad.untyped_storage().data_ptr()
            # an addition to 0.5 and one to the first pass's sum: a rounding each of what is there
            close(p.grad, 0.5 + (trial + 1) * q.double().cpu(), 0.5 + (trial + 1) * q.double().abs().cpu(), 3, "grad")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [2.0, 1.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_norm_adds_every_term_in_fp64(device, dtype, kind):
    """One large value in front of small ones in every 16 bytes: an fp32 sum of the terms would lose each of the small ones (0.9
    of half a step), together they are 1.35 steps of 2^-24 or more of the norm.  In fp64 the norm takes its last rounding only."""
    from jova_amd.train import clip_grad_norm_
    small = 0.9 * U32
    if dtype == torch.float16 and kind == 1.0:
        small = 2.0 ** -24                                           # (its least number: exactly half a step, a tie that goes to 1)
    v = torch.tensor(small if kind == 1.0 else small ** 0.5, dtype=torch.float64).to(dtype)
    assert float(v) > 0.0 and float(v) ** int(kind) <= U32
    x = torch.full((3, 16 // v.element_size()), 1.0, dtype=dtype)
    x[:, 1:] = v
    for n in (1, 3):
        for rows in (x[:n], x[:n].repeat(4096, 1)):                  # by single vectors and by whole chunks
            want = float(rows.double().norm(p=kind))
            got = float(clip_grad_norm_([rows.to(device)], 1e9, norm_type=kind))
            assert abs(got - want) <= U32 * want * (1 + 2.0 ** -20), (got, want)


@pytest.mark.gpu
def test_clipping_is_noticed_by_a_graph_that_saved_the_gradient(device):
    from jova_amd.train import clip_grad_norm_
    grads = [torch.full((5,), 2.0, device=device), torch.full((3,), 2.0, device=device).half()]
    outs = [torch.zeros_like(v) for v in grads]
    clip_grad_norm_(grads, 1.0, out=outs)
    assert [v._version for v in grads] == [0, 0] and all(v._version > 0 for v in outs)
    w = torch.ones(5, device=device, requires_grad=True)
    y = (w * grads[0]).sum()                                         # keeps grads[0] for w's gradient
    clip_grad_norm_(grads, 1.0)
    assert all(v._version > 0 for v in grads)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        v = torch.full((4,), 2.0, device=device)
        clip_grad_norm_([v], 1.0)
        assert abs(float(v.double().norm()) - 1.0) < 1e-5


class _Noted(torch.autograd.Function):
    """Stands for a differentiable call of the sequence functions (CPU)."""
    @staticmethod
    def forward(ctx, x, w):
        from jova_amd.nn import functional as F
        F._note_leaves(ctx, x, w)
        return x * w

    @staticmethod
    def backward(ctx, g):
        return g, g


def test_a_capture_over_a_graph_that_holds_the_leaves_by_other_functions_is_refused(monkeypatch):
    """Parameters behind a cast, an exponential or a product; accumulators that an earlier graph of another stream has made; graphs
    of other leaves are no hindrance, and nothing is kept of those that have ended, whatever thread made them."""
    import threading
    now = threading.local()
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now.stream, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capturing)
    x, w, other = torch.ones(2), torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True)

    def call(stream, w, capturing=False, before=lambda w: w, x=x):
        now.stream, now.capturing = stream, capturing
        return _Noted.apply(x, before(w))
    ways = [lambda w: w, lambda w: w.to(torch.bfloat16), lambda w: -torch.exp(w), lambda w: torch.nn.functional.relu(w * 2.0) + 1.0]
    for first in ways:
        for second in ways:
            eager = call(1, w, before=first)
            with pytest.raises(RuntimeError, match="eager graph"):
                call(2, w, True, second)
            kept = [call(2, other, True, second), call(2, other, True, second)]       # other leaves: twice, with the results alive
            del eager
            call(2, w, True, second)
            del kept
    # the accumulator of stream 1 lives on in a graph of stream 2, and in one that was built behind that
    old = call(1, w)
    new = call(2, w)
    del old
    newer = call(2, w)
    del new
    with pytest.raises(RuntimeError, match="eager graph"):
        call(2, w, True)
    call(2, other, True)
    del newer
    warm = call(2, w)
    call(2, w, True)                                                  # built on the capture's own stream
    del warm
    # a captured graph holds its leaves as an eager one does
    captured = call(2, w, True)
    with pytest.raises(RuntimeError, match="eager graph"):
        call(3, w, True)
    del captured
    from jova_amd.nn import functional as F
    assert not any(F._GRAPHS.values())

    def work(k):
        live = []
        for i in range(1500):
            live.append(call(10 + k, w))
            del live[:len(live) - k - i % 5]
    held = call(1, w)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    with pytest.raises(RuntimeError, match="eager graph"):
        call(2, w, True)
    del held
    assert not any(F._GRAPHS.values())


def test_objects_are_built_again_when_the_makefile_changes():
    """The flags stand in it: objects of other flags must not be linked with new ones."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jova_amd", "csrc")
    out = subprocess.run(["make", "-n", "-W", "Makefile", "-C", csrc], check=True, capture_output=True, text=True).stdout
    sources = sorted(f for f in os.listdir(csrc) if f.endswith(".hip"))
    compiled = [line for line in out.splitlines() if " -c " in line]
    assert len(sources) > 0 and all(any(" %s " % s in line for line in compiled) for s in sources), out


def test_the_scan_encoder_refuses_what_its_products_would_read_past_the_end():
    from jova_amd.nn.models import ProteinSSM
    net = ProteinSSM(6, 8, state_dim=4)
    x, st = torch.zeros(3, 2, 6), net.new_state(2, "cpu")
    with pytest.raises((RuntimeError, AssertionError)):
        net(x)                                                       # (fp32: as far as the products, which want a GPU)
    for bad in (x.bfloat16(), x.half(), x.double()):
        with pytest.raises(TypeError, match="float32"):
            net(bad)
        with pytest.raises(TypeError, match="float32"):
            net((bad, torch.tensor([3, 1])))
        with pytest.raises(TypeError, match="float32"):
            net.step(bad[0], st)
    with pytest.raises(ValueError, match="6 features"):
        net(x[..., :5])
    with pytest.raises(TypeError, match="float32"):
        net.bfloat16()(x.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 5])
def test_protein_words_of_every_type(device, dim, dtype):
    """Narrow tables too: the ids come from a kernel that reads a float a word."""
    from jova_amd.nn.models import ProteinWords
    rng = __import__("numpy").random.RandomState(5)
    prof = {"P%d" % i: rng.randint(0, 300, size=(n, 3)) for i, n in enumerate((4, 1, 9))}
    torch.manual_seed(2)
    words = ProteinWords(prof, 300, dim, scale=2.0).to(dtype).to(device)
    x, ln = words([("s", "P0"), ("s", "P1"), ("s", "P2")])
    assert ln.tolist() == [4, 1, 9] and x.dtype == dtype and x.shape == (9, 3, 3 * dim)
    w = words.embedding.weight.detach().double().cpu()
    want = torch.zeros(9, 3, 3 * dim, dtype=torch.float64)
    for i, k in enumerate(prof):
        want[:prof[k].shape[0], i] = (2.0 * w[torch.from_numpy(prof[k])]).reshape(-1, 3 * dim)
    assert torch.equal(x.detach().double().cpu(), want)              # (a doubling is exact)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,b,d,n,gr", [(700, 2, 132, 16, 2), (530, 3, 210, 32, 3), (780, 40, 260, 3, 2)])
def test_scan_chunks_and_pieces_with_groups_and_channel_tiles(device, t, b, d, n, gr, dtype):
    """A split time axis in every type, together with groups of several channel tiles (the last ones part empty) and ragged ends; in
    the last shape the backward pass's chunks are cut into pieces.  Roundings: scan_c, its derivation holds for any split, since
    a chunk's factor exp(A sum e) takes the place of as many products."""
    from jova_amd.nn import functional as F
    g = gen(t + b + d + n)
    a, dy, dh = scan_inputs(g, t, b, d, n, gr, dtype)
    lengths = torch.randint(0, t + 1, (b,), generator=g)
    lengths[:2] = torch.tensor([t, t // 2 + 5])
    keys = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")
    v = {k: a[k].to(device).requires_grad_(True) for k in keys}
    y, h = F.selective_scan(*(v[k] for k in keys[:8]), True, lengths.to(device), v["state"], True)
    got = dict(zip(keys, torch.autograd.grad((y, h), [v[k] for k in keys], (dy.to(device), dh.to(device)))))
    want, mag = (R.scan(*(a[k] for k in keys[:8]), True, lengths, a["state"], dy, dh, mag=m) for m in (False, True))
    c = scan_c(t, n)
    close(y, want[0], mag[0], c, "y")
    close(h, want[1], mag[1], c, "state")
    for k in keys:
        extra = {"A": t * b, "D": t * b, "bias": t * b, "B": d // gr, "C": d // gr}.get(k, 0)
        close(got[k], want[2][k], mag[2][k], 2 * c + extra, "d" + k)


@pytest.mark.gpu
def test_gradients_of_calls_on_another_stream_are_complete_behind_backward(device):
    """Forward passes on two streams, backward passes called from a third: the caller's stream waits for what they add to .grad."""
    from jova_amd.nn import functional as F
    g = gen(93)
    t, b, d, v = 2000, 8, 256, 500
    idx, dout = torch.randint(v, (t, b), generator=g).to(device), torch.randn(t, b, d, generator=g).to(device)
    params = [torch.randn(*s, generator=g).to(device).requires_grad_(True) for s in ((v, d), (d, 4), (d,))]

    def call():
        return F.causal_conv1d(F.embedding(idx, params[0]), params[1], params[2], "silu")
    want = torch.autograd.grad(call(), params, dout)
    for trial in range(5):
        for p in params:
            p.grad = torch.zeros_like(p)
        streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(call())
        for y in outs:
            y.backward(dout)
        assert all(torch.equal(p.grad, q + q) for p, q in zip(params, want)), trial
