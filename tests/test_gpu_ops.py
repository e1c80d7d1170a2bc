"""The operators around the MoE layer on the GPU, through the binding, against
plain implementations in 64 bits: dense INT4 products, residual norms, beam
selection and the reordering of states.

Tolerances come from the arithmetic, before any run.  EPS[t] / 2 is one
rounding to type t.  U = 2^-24 is one fp32 rounding.
"""
import ctypes as C

import numpy as np
import pytest

import llmoc_b200 as L

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def cuda_ready():
    assert torch.cuda.is_available(), "gpu tests need a CUDA device"
    yield
    torch.cuda.empty_cache()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def stream():
    return torch.cuda.current_stream()


def close(got, want, tol, what=""):
    """Elementwise |got - want| <= tol, all finite."""
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i}: {got[i].item()} for "
                             f"{want[i].item()}, tolerance {tol[i].item()}")


# ------------------------------------------------------------- INT4 products

class Weight:
    """Random QLWC weights on the device with their 64-bit matrix."""

    def __init__(self, M, K, gs, asym, seed, zp=7):
        g = gen(seed)
        ng = -(-K // gs)
        self.M, self.K, self.gs, self.asym = M, K, gs, asym
        self.q = torch.randint(0, 256, (M, K // 2), generator=g, device="cuda", dtype=torch.uint8)
        self.s = (torch.rand((M, ng), generator=g, device="cuda") * 0.02 + 0.001).half()
        self.z = (torch.randn((M, ng), generator=g, device="cuda") * 0.05).half() if asym else None
        self.view = L.view(self.q, self.s, self.z, M, K, gs, L.SCHEME_GPTQ_ASYM if asym else L.SCHEME_AWQ_SYM, zp)
        n = torch.stack([self.q & 15, self.q >> 4], 2).reshape(M, K).double()
        s = self.s.double().repeat_interleave(gs, 1)[:, :K]
        if asym:
            z = self.z.double().repeat_interleave(gs, 1)[:, :K]
            self.w, self.mag = n * s + z, n * s + z.abs()
        else:
            self.w = (n - zp) * s
            self.mag = self.w.abs()
        torch.cuda.synchronize()

    def tol(self, x, y, dtype):
        """One rounding to the output's type, plus the fp32 sums: a group's
        products are exact, each of its gs / 16 tensor-core steps and each of
        the ng (twice: scale and zero) + 8 later additions loses at most 4
        fp32 roundings of the magnitudes summed."""
        steps = self.gs / 16 + 2 * self.s.shape[1] + 8
        return y.abs() * (torch.finfo(dtype).eps / 2) + 4 * steps * U * (x.double().abs() @ self.mag.t())


def run_linear(lin, w, x, T, dtype, R=None, Y=None):
    Y = torch.full((T, w.M), float("nan"), dtype=dtype, device="cuda") if Y is None else Y
    lin.forward(x, T, Y, R=R, stream=stream())
    torch.cuda.synchronize()
    return Y


SHAPES = [  # M, K, group size
    (1, 32, 32), (15, 64, 32), (16, 96, 64), (17, 160, 128), (100, 224, 96), (48, 1024, 256), (2053, 416, 32),
    (333, 4128, 128), (4096, 2048, 128), (520, 1984, 64), (9000, 256, 128), (64, 16384, 32),
]


@pytest.mark.parametrize("M,K,gs", SHAPES)
@pytest.mark.parametrize("asym", [False, True])
def test_linear(M, K, gs, asym):
    w = Weight(M, K, gs, asym, seed=M + K)
    lin = L.Int4Linear.create([w.view], on_device=True)
    assert lin.weight_bytes() >= M * K // 2
    for T in (1, 2, 7, 8, 9, 16, 17, 31, 33, 70):
        x = torch.randn((T, K), generator=gen(T), device="cuda").to(BF16)
        r = torch.randn((T, M), generator=gen(T + 1), device="cuda").to(BF16)
        y = x.double() @ w.w.t()
        close(run_linear(lin, w, x, T, F32), y, w.tol(x, y, F32), f"T={T} fp32")
        yr = y + r.double()
        # the sum with the residual is one more fp32 addition
        close(run_linear(lin, w, x, T, BF16, R=r), yr, w.tol(x, yr, BF16) + 2 * U * (y.abs() + r.double().abs()),
              f"T={T} bf16 + residual")
    lin.close()


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("pad,off", [(1, 0), (8, 0), (3, 1), (24, 8)])
def test_linear_strides(T, pad, off):
    """Rows of any stride and alignment; what lies between Y's rows stays."""
    w = Weight(77, 192, 64, False, seed=3)
    lin = L.Int4Linear.create([w.view], on_device=True)
    big = torch.randn((T, w.K + pad + off), generator=gen(1), device="cuda").to(BF16)
    x = big[:, off:off + w.K]
    yb = torch.full((T, w.M + pad + off), 7.0, dtype=BF16, device="cuda")
    yv = yb[:, off:off + w.M]
    rb = torch.randn((T, w.M + pad), generator=gen(2), device="cuda").to(BF16)
    lin.forward(x, T, yv, R=rb[:, :w.M], stream=stream())
    torch.cuda.synchronize()
    y = x.double() @ w.w.t() + rb[:, :w.M].double()
    close(yv, y, w.tol(x, y, BF16) + 2 * U * (y.abs() + rb[:, :w.M].double().abs()))
    assert bool((yb[:, :off] == 7).all()) and bool((yb[:, off + w.M:] == 7).all())


def test_linear_in_place_residual_and_shared_buffer():
    w = Weight(192, 192, 64, True, seed=4)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((9, 192), generator=gen(5), device="cuda").to(BF16)
    r = torch.randn((9, 192), generator=gen(6), device="cuda").to(BF16)
    want = run_linear(lin, w, x, 9, BF16, R=r)
    both = r.clone()
    lin.forward(x, 9, both, R=both, stream=stream())
    wide = torch.zeros((9, 384), dtype=BF16, device="cuda")  # X and Y as columns of one buffer
    wide[:, :192] = x
    lin.forward(wide[:, :192], 9, wide[:, 192:], R=r, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(both, want) and torch.equal(wide[:, 192:], want)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("on_device", [False, True])
def test_linear_stacked_views(asym, on_device):
    """Projections that share their input, stacked; host and device buffers; a group left over at the end of K."""
    ws = [Weight(m, 352, 64, asym, seed=m) for m in (48, 16, 37)]
    host = [(w.q.cpu().numpy(), w.s.cpu().numpy(), w.z.cpu().numpy() if asym else None) for w in ws]
    views = [w.view if on_device else L.view(*h, w.M, w.K, w.gs, 1 if asym else 2) for w, h in zip(ws, host)]
    lin = L.Int4Linear.create(views, on_device=on_device)
    assert (lin.M, lin.K) == (101, 352)
    x = torch.randn((6, 352), generator=gen(8), device="cuda").to(BF16)
    y = torch.empty((6, 101), dtype=F32, device="cuda")
    lin.forward(x, 6, y, stream=stream())
    torch.cuda.synchronize()
    at = 0
    for w in ws:
        want = x.double() @ w.w.t()
        close(y[:, at:at + w.M], want, w.tol(x, want, F32))
        at += w.M


@pytest.mark.parametrize("zp", [1, 8, 15, 20, 127])
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("T", [3, 20, 70])
def test_linear_zero_points(zp, gs, T):
    w = Weight(40, 384, gs, False, seed=zp, zp=zp)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T, 384), generator=gen(9), device="cuda").to(BF16)
    y = x.double() @ w.w.t()
    # the group sums hold (16 + q) x: their roundings are those of at most 31 |x| s where the weights are smaller
    s = w.s.double().repeat_interleave(gs, 1)[:, :384]
    tol = w.tol(x, y, F32) + 8 * U * (x.double().abs() @ (31 * s).t())
    close(run_linear(lin, w, x, T, F32), y, tol)
    lin.status(stream())


@pytest.mark.parametrize("T", [3, 12, 40])
def test_linear_non_finite_rows_stay_apart(T):
    """A token with inf or NaN changes no other token's bits."""
    w = Weight(200, 512, 128, False, seed=11)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T, 512), generator=gen(10), device="cuda").to(BF16)
    clean = run_linear(lin, w, x, T, F32)
    x[1, 100] = float("inf")
    x[T - 1, 3] = float("nan")
    y = run_linear(lin, w, x, T, F32)
    keep = [t for t in range(T) if t not in (1, T - 1)]
    assert torch.equal(y[keep], clean[keep])
    assert not bool(torch.isfinite(y[1, (w.w[:, 100] != 0)]).any()) and bool(torch.isnan(y[T - 1]).all())


def test_linear_same_bits_and_empty_batch():
    """Two calls give the same bits; T = 0 writes nothing."""
    w = Weight(1000, 2048, 128, False, seed=12)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((5, 2048), generator=gen(13), device="cuda").to(BF16)
    a, b = run_linear(lin, w, x, 5, F32), run_linear(lin, w, x, 5, F32)
    assert torch.equal(a, b)
    y = torch.full((5, 1000), 3.0, dtype=F32, device="cuda")
    lin.forward(x, 0, y, stream=stream())
    torch.cuda.synchronize()
    assert bool((y == 3).all())


# --------------------------------------------------------------------- norms

E = 64 * U  # a row's reduction (at most 32 values a thread, 5 + 16 steps) and the roundings around it


def ref_normed(x, err, kind, w, b, off, eps):
    """(norm, error bound) of x whose elements carry an error of at most err."""
    if kind == "none":
        return x, err
    if kind == "layer":
        mean = x.mean(1, keepdim=True)
        err = err + err.mean(1, keepdim=True) + E * (x.abs() + x.abs().mean(1, keepdim=True))
        x = x - mean
    rms = ((x * x).mean(1, keepdim=True) + eps).sqrt()
    rel = E + err.pow(2).mean(1, keepdim=True).sqrt() / rms  # of the root
    wd = 1.0 if w is None else w.double() + off
    n = x / rms * wd
    err = n.abs() * rel + err / rms * (abs(wd) if w is None else wd.abs()) + E * n.abs()
    if b is not None:
        n = n + b.double()
        err = err + E * b.double().abs()
    return n, err


def ref_norm(block, res, gate, c):
    r, err = torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros((), dtype=torch.float64, device="cuda")
    if res is not None:
        r = c["residual_scale"] * res.double()
        err = 2 * U * r.abs()
    if block is not None:
        x = block.double()
        u, eu = ref_normed(x, torch.zeros_like(x), c["post"], c["post_weight"], c["post_bias"], c["weight_offset"],
                           c["eps"])
        g = torch.ones((), dtype=torch.float64, device="cuda")
        if gate is not None:
            g = gate.double()
            g = torch.sigmoid(g) if c["gate_act"] == "sigmoid" else g
        v = c["block_scale"] * g * u
        err = err + (c["block_scale"] * g).abs() * eu + E * v.abs() + 2 * U * (r.abs() + v.abs())
        r = r + v
    n, en = ref_normed(r, err + torch.zeros_like(r), c["pre"], c["pre_weight"], c["pre_bias"], c["weight_offset"],
                       c["eps"])
    return r, err, n, en


def norm_config(H, post, pre, wdt, seed, **kw):
    g = gen(seed)

    def vec(mean):
        return (torch.randn((H,), generator=g, device="cuda") * 0.3 + mean).to(wdt)

    c = dict(post=post, pre=pre, post_weight=vec(1) if post != "none" else None,
             post_bias=vec(0) if post == "layer" else None, pre_weight=vec(1) if pre != "none" else None,
             pre_bias=vec(0) if pre == "layer" else None, weight_offset=0.0, eps=1e-5, block_scale=0.7,
             residual_scale=1.25, gate_act="none")
    c.update(kw)
    return c


def check_rows(got, want, err, what):
    close(got, want, err + want.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 2.0 ** -8), what)


@pytest.mark.parametrize("H", [1, 2, 7, 8, 255, 256, 257, 1000, 1024, 1032, 2048, 2050, 4096, 4104, 5001, 8192, 8200,
                               16383, 16384])
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("rms", "rms"), ("layer", "layer"), ("rms", "none")])
def test_norm(H, post, pre):
    for T, rdt, bdt, ndt, wdt in ((1, BF16, BF16, BF16, BF16), (5, F32, BF16, BF16, F32), (3, F32, F32, F32, BF16)):
        c = norm_config(H, post, pre, wdt, seed=H)
        op = L.ResidualNorm(H, **c)
        g = gen(T)
        b = (torch.randn((T, H), generator=g, device="cuda") * 2 + 0.5).to(bdt)
        r = (torch.randn((T, H), generator=g, device="cuda") * 3 - 0.25).to(rdt)
        ro, no = torch.empty_like(r), torch.empty((T, H), dtype=ndt, device="cuda")
        op.forward(T, b, r, ro, no, stream=stream())
        torch.cuda.synchronize()
        wr, er, wn, en = ref_norm(b, r, None, c)
        check_rows(ro, wr, er, f"T={T} residual")
        check_rows(no, wn, en, f"T={T} norm")


@pytest.mark.parametrize("H", [96, 515, 3000, 6144])
@pytest.mark.parametrize("gate,act", [((7, 1), "sigmoid"), ((1, 0), "none"), ((7, 0), "sigmoid"), ((1, 1), "none")])
@pytest.mark.parametrize("gdt", [BF16, F32])
def test_norm_gates(H, gate, act, gdt):
    """One gate per token, per channel, per element, or one for all."""
    T = 7
    c = norm_config(H, "rms", "layer", BF16, seed=H, gate_act=act, weight_offset=1.0, residual_scale=1.0)
    op = L.ResidualNorm(H, **c)
    b = torch.randn((T, H), generator=gen(1), device="cuda").to(BF16)
    r = torch.randn((T, H), generator=gen(2), device="cuda").to(BF16)
    gt = (torch.randn((gate[0], gate[1] or H), generator=gen(3), device="cuda") * 2).to(gdt)
    ro, no = torch.empty_like(r), torch.empty_like(b)
    op.forward(T, b, r, ro, no, gate=gt, stream=stream())
    torch.cuda.synchronize()
    wr, er, wn, en = ref_norm(b, r, gt, c)
    check_rows(ro, wr, er, "residual")
    check_rows(no, wn, en, "norm")


@pytest.mark.parametrize("H,pad", [(64, 8), (64, 3), (2048, 8), (2048, 5), (5000, 16)])
def test_norm_strides_and_partial_operands(H, pad):
    """Strided rows; no block (a plain norm), no residual, one output alone; in place."""
    T = 133
    c = norm_config(H, "layer", "rms", F32, seed=H)
    op = L.ResidualNorm(H, **c)

    def rows(seed, dt):
        return (torch.randn((T, H + pad), generator=gen(seed), device="cuda") * 2).to(dt)[:, :H]

    b, r = rows(1, BF16), rows(2, BF16)
    out = torch.full((T, H + pad), 9.0, dtype=BF16, device="cuda")
    no = out[:, :H]
    op.forward(T, None, r, None, no, stream=stream())
    torch.cuda.synchronize()
    _, _, wn, en = ref_norm(None, r, None, c)
    check_rows(no, wn, en, "plain norm")
    assert bool((out[:, H:] == 9).all())
    op.forward(T, b, None, None, no, stream=stream())
    torch.cuda.synchronize()
    _, _, wn, en = ref_norm(b, None, None, c)
    check_rows(no, wn, en, "no residual")
    wr, er, wn, en = ref_norm(b, r, None, c)
    b2, r2 = b.clone(), r.clone()
    op.forward(T, b2, r2, r2, b2, stream=stream())  # the residual stream in place, the block's buffer reused
    torch.cuda.synchronize()
    check_rows(r2, wr, er, "in place")
    check_rows(b2, wn, en, "in place norm")
    r3 = torch.empty_like(r2)
    op.forward(T, b, r, r3, None, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(r3, r2)


def test_norm_special_rows():
    """A zero row stays zero under RMS norm; a row with an infinity or NaN changes no other."""
    H, T = 1500, 6
    c = norm_config(H, "none", "rms", BF16, seed=1, residual_scale=1.0)
    op = L.ResidualNorm(H, **c)
    r = torch.randn((T, H), generator=gen(1), device="cuda").to(BF16)
    r[2] = 0
    clean, no = torch.empty_like(r), torch.empty_like(r)
    op.forward(T, None, r, None, clean, stream=stream())
    r[4, 7] = float("inf")
    r[5, 9] = float("nan")
    op.forward(T, None, r, None, no, stream=stream())
    torch.cuda.synchronize()
    assert bool((no[2] == 0).all()) and torch.equal(no[:4], clean[:4])
    assert bool(torch.isnan(no[4, 7])) and bool(torch.isnan(no[5]).all())
    big = torch.full((1, H), 1e18, dtype=F32, device="cuda")  # the squares sum far from overflow's edge
    out = torch.empty((1, H), dtype=F32, device="cuda")
    op.forward(1, None, big, None, out, stream=stream())
    torch.cuda.synchronize()
    want = c["pre_weight"].double()[None]
    close(out, want, E * 2 * want.abs())


@pytest.mark.parametrize("H", [200, 3000])
def test_norm_large_values(H):
    """Rows whose sums or squares leave fp32's range, a constant one among them."""
    x = torch.randn((4, H), generator=gen(H), device="cuda")
    x[0] *= 1e25
    x[1] = x[1] * 1e30 + 3e37
    x[2] = 2e37
    x[3] *= 1e-18
    for kind in ("rms", "layer"):
        c = norm_config(H, "none", kind, F32, seed=2, residual_scale=1.0)
        out = torch.empty((4, H), dtype=F32, device="cuda")
        L.ResidualNorm(H, **c).forward(4, None, x, None, out, stream=stream())
        torch.cuda.synchronize()
        _, _, wn, en = ref_norm(None, x, None, c)
        if kind == "layer":  # the mean of equal values, and so the row, is exact to E of the values
            near = (out[2].double() - c["pre_bias"].double()).abs() / c["pre_weight"].double().abs()
            assert bool((near <= 1.01).all()) and not bool(torch.isnan(out).any())
            keep = [0, 1, 3]
            out, wn, en = out[keep], wn[keep], en[keep]
        close(out, wn, en + wn.abs() * U, kind)


# --------------------------------------------------------------- beam search

def ref_select(logits, scores, fin, eos, k):
    """Plain selection in 64 bits; ties to the lowest beam, then token."""
    B, W = scores.shape
    V = logits.shape[1]
    ninf = float("-inf")
    x = logits.double()
    x = torch.where(torch.isfinite(x), x, ninf)
    sc = scores.double()
    sc = torch.where(torch.isfinite(sc), sc, ninf)
    cand = sc.reshape(B * W, 1) + x - torch.logsumexp(x, 1, keepdim=True)
    cand = torch.where(x > ninf, cand, ninf).reshape(B, W, V)
    if fin is not None:
        stay = torch.full((B, W, V), ninf, dtype=torch.float64, device=x.device)
        stay[:, :, eos] = sc
        cand = torch.where(fin.bool()[..., None], stay, cand)
    cand = torch.where(torch.isnan(cand), ninf, cand).reshape(B, W * V)
    v, i = torch.sort(cand, dim=1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k]
    if v.shape[1] < k:
        v = torch.nn.functional.pad(v, (0, k - v.shape[1]), value=ninf)
        i = torch.nn.functional.pad(i, (0, k - i.shape[1]))
    live = v > ninf
    parent, token = torch.where(live, i // V, -1), torch.where(live, i % V, -1)
    f = live & (token == eos)
    if fin is not None:
        f = f | (live & fin.bool().gather(1, parent.clamp_min(0)))
    return parent, token, v, f


def run_select(logits, scores, fin, eos, k, want_fin=True, ws=None):
    B, W = scores.shape
    bs = L.BeamSearch(B, W, logits.shape[1], k, eos_token=eos)
    n = bs.workspace_bytes()
    if ws is None:
        ws = torch.randint(0, 256, (n,), device="cuda", dtype=torch.uint8)  # whatever it holds
    parent = torch.full((B, k), 77, dtype=torch.int32, device="cuda")
    token, out = parent.clone(), torch.full((B, k), 77.0, device="cuda")
    fo = torch.full((B, k), 77, dtype=torch.uint8, device="cuda") if want_fin else None
    bs.select(logits, scores, parent, token, out, ws, n, finished=fin, finished_out=fo, stream=stream())
    torch.cuda.synchronize()
    return parent, token, out, fo


def check_select(logits, scores, fin, eos, k):
    parent, token, out, fo = run_select(logits, scores, fin, eos, k)
    wp, wt, wv, wf = ref_select(logits, scores, fin, eos, k)
    assert torch.equal(parent.long(), wp), (parent, wp)
    assert torch.equal(token.long(), wt), (token, wt)
    assert torch.equal(fo.bool(), wf)
    live = wv > float("-inf")
    assert bool((out[~live] == float("-inf")).all())
    # the log-sum: exponentials within 4 fp32 roundings and |x - max| of another, at most 32 + 16 additions; the
    # value's own rounding
    tol = 200 * U + wv.abs() * U
    close(out[live], wv[live], tol[live], "scores")


@pytest.mark.parametrize("V", [1, 2, 31, 256, 2047, 2048, 2049, 8193, 40000, 70001])
@pytest.mark.parametrize("B,W,k", [(1, 1, 1), (1, 4, 4), (3, 5, 10), (17, 8, 8)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_select(V, B, W, k, dt):
    g = gen(V + 10 * W)
    logits = (torch.randn((B * W, V), generator=g, device="cuda") * 3).to(dt)
    scores = -20 * torch.rand((B, W), generator=g, device="cuda")
    check_select(logits, scores, None, -1, k)
    fin = (torch.rand((B, W), generator=g, device="cuda") < 0.4).to(torch.uint8)
    check_select(logits, scores, fin, V // 2, k)


@pytest.mark.parametrize("W,k", [(16, 32), (128, 128), (3, 100), (1, 17), (2, 65)])
def test_select_many_candidates(W, k):
    g = gen(W + k)
    logits = (torch.randn((2 * W, 3001), generator=g, device="cuda")).to(BF16)
    check_select(logits, -torch.rand((2, W), generator=g, device="cuda"), None, 5, k)


@pytest.mark.parametrize("pattern", ["equal", "ascending", "descending", "one_group", "two_values", "zeros"])
@pytest.mark.parametrize("V", [700, 20011])
@pytest.mark.parametrize("k", [4, 24])
def test_select_ties_and_orders(pattern, V, k):
    """Values that defeat the bound (far more elements reach it than are
    wanted), ties inside a beam, and beams that are equal throughout."""
    i = torch.arange(V, device="cuda", dtype=torch.float32)
    row = {"equal": torch.full((V,), 1.5, device="cuda"), "ascending": i / V, "descending": -i / V,
           "one_group": torch.where((i >= 256) & (i < 1500), 5 + i % 7, -i / V), "two_values": (i % 2),
           "zeros": torch.where(i % 3 == 0, -0.0, 0.0)}[pattern]
    for dt in (BF16, F32):
        logits = row.to(dt).expand(6, V).contiguous()
        check_select(logits, torch.zeros((2, 3), device="cuda"), None, 1, k)
    logits = row.expand(256, V).contiguous()  # more tied lists than the merge's list holds
    check_select(logits, torch.full((2, 128), -2.0, device="cuda"), None, 1, k)


@pytest.mark.parametrize("V", [50, 9001])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_select_masks(V, dt):
    """Rows with nothing left, one token left, NaN and infinities, lowest
    values, dead and finished beams; fewer candidates than wanted."""
    inf, low = float("inf"), torch.finfo(dt).min
    B, W, k = 5, 4, 6
    x = torch.randn((B, W, V), generator=gen(V), device="cuda").to(dt)
    x[0, :, :] = -inf                       # a sequence without any candidate
    x[1, 0] = -inf
    x[1, 0, V - 1] = 2                      # one token left
    x[1, 1:] = float("nan")
    x[2, 0, ::2] = inf                      # masked, not dominant
    x[2, 1] = low                           # every token at the type's lowest value: uniform
    x[3, 0] = low
    x[3, 0, 3] = 0.5
    scores = -torch.rand((B, W), generator=gen(1), device="cuda")
    scores[3, 1:] = torch.tensor([-inf, inf, float("nan")], device="cuda")
    scores[4, 1:] = -inf
    fin = torch.zeros((B, W), dtype=torch.uint8, device="cuda")
    check_select(x.reshape(B * W, V), scores, fin, 0, k)
    fin[0, 2] = 1
    fin[3, 1] = 1                           # finished, but dead
    fin[4, 0] = 7
    check_select(x.reshape(B * W, V), scores, fin, V - 1, k)


def test_select_strides_and_no_finished_out():
    g = gen(3)
    for pad, off, dt in ((1, 0, BF16), (8, 8, BF16), (5, 3, F32), (4, 4, F32)):
        big = torch.randn((6, 5000 + pad + off), generator=g, device="cuda").to(dt)
        x = big[:, off:off + 5000]
        scores = -torch.rand((2, 3), generator=g, device="cuda")
        parent, token, out, _ = run_select(x, scores, None, -1, 6, want_fin=False)
        wp, wt, _, _ = ref_select(x, scores, None, -1, 6)
        assert torch.equal(parent.long(), wp) and torch.equal(token.long(), wt)


# ------------------------------------------------------------------- reorder

@pytest.mark.parametrize("row", [1, 2, 15, 16, 100, 1001, 4096, 70000])
@pytest.mark.parametrize("B,W,k", [(1, 4, 4), (3, 5, 7), (2, 16, 16), (2, 40, 33), (1, 64, 64)])
def test_reorder(row, B, W, k):
    g = gen(row + W)
    src = [torch.randint(0, 256, (B, W, row), generator=g, device="cuda", dtype=torch.uint8) for _ in range(3)]
    dst = [torch.full((B, k, row), 0xAB, device="cuda", dtype=torch.uint8) for _ in range(3)]
    parent = torch.randint(0, W, (B, k), generator=g, device="cuda", dtype=torch.int32)
    parent[0, 0] = -1
    parent[-1, -1] = W
    L.BeamReorder(src, dst, B, W, k).run(parent, stream=stream())
    torch.cuda.synchronize()
    ok = (parent >= 0) & (parent < W)
    for s, d in zip(src, dst):
        want = torch.full_like(d, 0xAB)
        got = s[torch.arange(B, device="cuda")[:, None], parent.long().clamp(0, W - 1)]
        want[ok] = got[ok]
        assert torch.equal(d, want)


@pytest.mark.parametrize("W", [1, 3, 8, 17, 32, 64])
@pytest.mark.parametrize("shape", [(7,), (4, 30, 16), (3, 50)])
def test_reorder_in_place(W, shape):
    """A permutation with repeats in place; rows with no parent, and what lies past the used length, stay."""
    B = 3
    src = [torch.randn((B, W) + shape, generator=gen(W + i), device="cuda").to(dt) for i, dt in enumerate((F32, BF16))]
    was = [s.clone() for s in src]
    parent = torch.randint(0, W, (B, W), generator=gen(W), device="cuda", dtype=torch.int32)
    parent[1, W // 2] = -1
    dim = len(shape) - 2 if len(shape) > 1 else 0
    used = shape[dim] * 2 // 3
    op = L.BeamReorder(src, src, B, W, W, dim=dim, used=used)
    op.run(parent, stream=stream())
    torch.cuda.synchronize()
    ok = parent >= 0
    for s, w in zip(src, was):
        full = w[torch.arange(B, device="cuda")[:, None], parent.long().clamp_min(0)]
        full[~ok] = w[~ok]
        want = w.clone()
        sel = [slice(None)] * (2 + dim) + [slice(0, used)]
        want[tuple(sel)] = full[tuple(sel)]
        assert torch.equal(s, want)


def test_reorder_many_tensors_and_unaligned():
    """More tensors than one launch takes, rows at odd addresses, an empty tensor among them."""
    B, W = 2, 4
    flat = torch.randint(0, 256, (130, 3 + B * W * 37), generator=gen(1), device="cuda", dtype=torch.uint8)
    src = [flat[i, i % 4:i % 4 + B * W * 37].view(B, W, 37) for i in range(130)]
    out = torch.zeros((130, B, W, 37), device="cuda", dtype=torch.uint8)
    dst = [out[i] for i in range(130)]
    parent = torch.tensor([[3, 3, 0, 1], [2, 0, 0, 2]], device="cuda", dtype=torch.int32)
    n0 = L.launch_count()
    L.BeamReorder(src, dst, B, W, W).run(parent, stream=stream())
    torch.cuda.synchronize()
    assert L.launch_count() - n0 == 3
    for s, d in zip(src, dst):
        assert torch.equal(d, s[torch.arange(B, device="cuda")[:, None], parent.long()])


def test_reorder_time_major_segments():
    """Rows interleaved in a time-major cache: segments further apart than rows."""
    B, W, steps, d = 2, 3, 11, 24
    cache = torch.randint(0, 256, (steps, B * W, d), generator=gen(2), device="cuda", dtype=torch.uint8)
    was = cache.clone()
    parent = torch.tensor([[1, 1, 0], [2, 2, 1]], device="cuda", dtype=torch.int32)
    t = (L.ReorderTensor * 1)(L.ReorderTensor(cache.data_ptr(), cache.data_ptr(), d, d, B * W * d, d, 9))
    L.check(L.lib.llmoc_beam_reorder(t, 1, parent.data_ptr(), B, W, W, 0, stream().cuda_stream), "reorder")
    torch.cuda.synchronize()
    rows = (parent.long() + torch.arange(B, device="cuda")[:, None] * W).reshape(-1)
    want = was.clone()
    want[:9] = was[:9][:, rows]
    assert torch.equal(cache, want)


# ------------------------------------------------------- the operators together

def moe_layer(oracle, seed=5, H=512, **kw):
    import orc

    rng = np.random.default_rng(seed)
    return L.MoeLayer.from_host(orc.make_layer(oracle, rng, H=H, I=256, E=16, topk=4, gs=128, **kw), 0)


@pytest.mark.parametrize("T", [1, 6, 40])
def test_moe_block_is_its_three_calls(oracle, T):
    """llmoc_moe_forward_block gives the bits of norm, layer and residual norm called one by one, in place or not."""
    layer = moe_layer(oracle)
    H = 512
    before = L.ResidualNorm(H, **norm_config(H, "rms", "rms", BF16, 1))
    after = L.ResidualNorm(H, **norm_config(H, "layer", "rms", BF16, 2, gate_act="sigmoid"))
    plain = L.ResidualNorm(H, pre="rms", pre_weight=before._keep[1], eps=1e-5)
    r = torch.randn((T, H), generator=gen(1), device="cuda").to(BF16)
    gate = torch.randn((T, 1), generator=gen(2), device="cuda").to(BF16)
    x, b, ro, no = (torch.empty_like(r) for _ in range(4))
    n = layer.block_workspace_bytes(T)
    ws = torch.empty((n,), dtype=torch.uint8, device="cuda")
    plain.forward(T, None, r, None, x, stream=stream())
    layer.forward(x, T, b, ws, layer.workspace_bytes(T), stream())
    after.forward(T, b, r, ro, no, gate=gate, stream=stream())
    ro2, no2 = torch.empty_like(r), torch.empty_like(r)
    layer.forward_block(before, after, T, r, ro2, no2, ws, n, gate=gate, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(ro, ro2) and torch.equal(no, no2)
    r2 = r.clone()
    layer.forward_block(before, after, T, r2, r2, None, ws, n, gate=gate, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(r2, ro)
    with pytest.raises(L.LlmocError, match="WORKSPACE"):
        layer.forward_block(before, after, T, r, ro2, no2, ws, n - 1, gate=gate, stream=stream())
    layer.close()


class Step:
    """A decode step of a toy decoder: a MoE block, the final norm in its tail,
    an INT4 head with fp32 logits, the beams' selection, their states moved."""

    def __init__(self, oracle, batch=2, beams=4, vocab=1500, H=512):
        self.batch, self.beams, self.H, self.vocab = batch, beams, H, vocab
        T = self.T = batch * beams
        self.layer = moe_layer(oracle)
        self.before = L.ResidualNorm(H, **norm_config(H, "none", "rms", BF16, 1))
        self.c = norm_config(H, "rms", "rms", BF16, 2)
        self.after = L.ResidualNorm(H, **self.c)
        self.head_w = Weight(vocab, H, 128, False, seed=3)
        self.head = L.Int4Linear.create([self.head_w.view], on_device=True)
        self.beam = L.BeamSearch(batch, beams, vocab, beams, eos_token=7)
        self.ws = torch.empty((self.layer.block_workspace_bytes(T),), dtype=torch.uint8, device="cuda")
        self.bws = torch.empty((self.beam.workspace_bytes(),), dtype=torch.uint8, device="cuda")
        self.r = torch.zeros((T, H), dtype=BF16, device="cuda")
        self.h, self.ro = torch.empty_like(self.r), torch.empty_like(self.r)
        self.logits = torch.empty((T, vocab), dtype=F32, device="cuda")
        self.scores = torch.zeros((batch, beams), device="cuda")
        self.fin = torch.zeros((batch, beams), dtype=torch.uint8, device="cuda")
        self.parent = torch.empty((batch, beams), dtype=torch.int32, device="cuda")
        self.token, self.out = torch.empty_like(self.parent), torch.empty_like(self.scores)
        self.fin_out = torch.empty_like(self.fin)
        self.states = [torch.zeros((batch, beams, 6, 40), dtype=BF16, device="cuda") for _ in range(5)]
        self.move = L.BeamReorder(self.states, self.states, batch, beams, beams)

    def set(self, seed):
        g = gen(seed)
        self.r.copy_(torch.randn(self.r.shape, generator=g, device="cuda"))
        self.scores.copy_(-5 * torch.rand(self.scores.shape, generator=g, device="cuda"))
        self.fin.copy_(torch.rand(self.fin.shape, generator=g, device="cuda") < 0.2)
        for s in self.states:
            s.copy_(torch.randn(s.shape, generator=g, device="cuda"))

    def run(self, st):
        self.layer.forward_block(self.before, self.after, self.T, self.r, self.ro, self.h, self.ws, self.ws.numel(),
                                 stream=st)
        self.head.forward(self.h, self.T, self.logits, stream=st)
        self.beam.select(self.logits, self.scores, self.parent, self.token, self.out, self.bws, self.bws.numel(),
                         finished=self.fin, finished_out=self.fin_out, stream=st)
        self.move.run(self.parent, stream=st)

    def check(self, was):
        y = self.h.double() @ self.head_w.w.t()
        close(self.logits, y, self.head_w.tol(self.h, y, F32), "logits")
        wp, wt, wv, wf = ref_select(self.logits, self.scores, self.fin, 7, self.beams)
        assert torch.equal(self.parent.long(), wp) and torch.equal(self.token.long(), wt)
        assert torch.equal(self.fin_out.bool(), wf)
        rows = torch.arange(self.batch, device="cuda")[:, None]
        for s, w in zip(self.states, was):
            assert torch.equal(s, w[rows, self.parent.long()])


def test_decode_step_on_a_side_stream(oracle):
    s = Step(oracle)
    side = torch.cuda.Stream()
    for seed in range(3):
        s.set(seed)
        was = [x.clone() for x in s.states]
        side.wait_stream(torch.cuda.current_stream())
        s.run(side)
        side.synchronize()
        s.check(was)


def test_decode_step_captured(oracle):
    """The step in a CUDA graph, replayed on new inputs; two graphs with workspaces of their own interleaved."""
    a, b = Step(oracle), Step(oracle, batch=3, beams=2, vocab=9001)
    graphs = []
    for s in (a, b):
        s.set(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        s.run(side)  # once before the capture
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.run(torch.cuda.current_stream())
        graphs.append(g)
    for seed in range(4, 7):
        was = []
        for s in (a, b):
            s.set(seed)
            was.append([x.clone() for x in s.states])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        a.check(was[0])
        b.check(was[1])


# ------------------------------------------------------------------ refusals

def test_binding_refuses_wrong_tensors():
    w = Weight(32, 64, 32, False, seed=1)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x, y = torch.zeros((4, 64), dtype=BF16, device="cuda"), torch.full((4, 32), 5.0, dtype=F32, device="cuda")
    bad = [(x.cpu(), y, None), (x.float(), y, None), (x, y.half(), None), (x[:, ::2], y, None), (x[:, :32], y, None),
           (x, y[:, :16], None), (x, y[:3], None), (x, y, x[:, :32].float()), (x.t(), y, None)]
    for xx, yy, rr in bad:
        with pytest.raises(L.LlmocError):
            lin.forward(xx, 4, yy, R=rr, stream=stream())
    with pytest.raises(L.LlmocError, match="overlaps"):
        buf = torch.zeros((4, 64), dtype=BF16, device="cuda")
        lin.forward(buf, 4, buf[:, :32], stream=stream())
    with pytest.raises(L.LlmocError, match="overlaps"):
        buf = torch.zeros((5, 32), dtype=BF16, device="cuda")
        lin.forward(x, 4, buf[1:], R=buf[:4], stream=stream())
    lin.close()
    with pytest.raises(L.LlmocError):
        lin.forward(x, 4, y, stream=stream())
    op = L.ResidualNorm(64, pre="rms")
    for args in ((4, None, x.half(), None, x), (4, None, x, None, x[:, :32]), (4, x, x.float(), x, None),
                 (4, x.cpu(), x, None, x), (5, None, x, None, x.clone())):
        with pytest.raises(L.LlmocError):
            op.forward(*args, stream=stream())
    bs = L.BeamSearch(1, 4, 64, 4)
    i = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    sc = torch.zeros((1, 4), device="cuda")
    ws = torch.empty((bs.workspace_bytes(),), dtype=torch.uint8, device="cuda")
    for args in ((x[:3], sc, i, i.clone(), sc.clone(), ws, ws.numel()), (x, sc, i, i, sc.clone(), ws, ws.numel()),
                 (x, sc, i, i.clone(), sc, ws, ws.numel()), (x, sc, i.long(), i, sc.clone(), ws, ws.numel()),
                 (x, sc, i, i.clone(), sc.clone(), ws, ws.numel() - 1), (x.half(), sc, i, i.clone(), sc.clone(), ws, ws.numel())):
        with pytest.raises(L.LlmocError):
            bs.select(*args, stream=stream())
    s = torch.zeros((2, 4, 8), device="cuda")
    with pytest.raises(L.LlmocError):
        L.BeamReorder([s], [torch.zeros((2, 4, 7), device="cuda")], 2, 4, 4)
    with pytest.raises(L.LlmocError):
        L.BeamReorder([s], [s.half()], 2, 4, 4)
    flat = torch.zeros((3, 4, 8), device="cuda")
    with pytest.raises(L.LlmocError, match="overlaps"):
        L.BeamReorder([flat[:2]], [flat[1:]], 2, 4, 4).run(torch.zeros((2, 4), dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert bool((y == 5).all()) and bool((s == 0).all())


# --------------------------------------------- shapes and calls at the edges

@pytest.mark.parametrize("M,K,gs", [(130, 640, 32), (300, 1408, 64), (300, 1376, 32), (700, 896, 128), (129, 2944, 128)])
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("pad", [0, 8, 5])
def test_linear_k_split_at_odd_steps(M, K, gs, asym, pad):
    """An odd number of 128-wide steps over several CTAs, aligned and unaligned
    rows, one to three blocks of tokens."""
    w = Weight(M, K, gs, asym, seed=M + K + gs)
    lin = L.Int4Linear.create([w.view], on_device=True)
    for T in (9, 12, 20, 48, 64, 65, 150):
        x = torch.randn((T, K + pad), generator=gen(T), device="cuda").to(BF16)[:, :K]
        y = x.double() @ w.w.t()
        got = run_linear(lin, w, x, T, F32)
        close(got, y, w.tol(x, y, F32), f"T={T}")
        assert torch.equal(got, run_linear(lin, w, x, T, F32))
    lin.status(stream())
    lin.close()


@pytest.mark.parametrize("T", [1, 8, 16, 30])
@pytest.mark.parametrize("gs", [32, 128])
def test_linear_on_two_streams_at_once(T, gs):
    """One handle, two streams: each call its own answer."""
    w = Weight(6000, 1024, gs, True, seed=21)
    lin = L.Int4Linear.create([w.view], on_device=True)
    xs = [torch.randn((T, w.K), generator=gen(i), device="cuda").to(BF16) for i in range(2)]
    want = [run_linear(lin, w, x, T, F32) for x in xs]
    st = [torch.cuda.Stream() for _ in range(2)]
    ys = [[torch.empty((T, w.M), device="cuda") for _ in range(10)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(10):
        for j in range(2):
            lin.forward(xs[j], T, ys[j][i], stream=st[j])
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(y, want[j]) for y in ys[j])
    lin.status(stream())


@pytest.mark.parametrize("T", [1, 7, 12, 40])
def test_rows_past_the_last_stay(T):
    """Buffers with more rows than the call: the others keep their bits."""
    w = Weight(200, 256, 32, False, seed=31)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T + 9, w.K), generator=gen(1), device="cuda").to(BF16)
    x[T:] = float("nan")
    y = torch.full((T + 9, w.M), 5.0, dtype=BF16, device="cuda")
    lin.forward(x, T, y, stream=stream())
    op = L.ResidualNorm(w.K, pre="rms")
    r = torch.randn((T + 9, w.K), generator=gen(2), device="cuda").to(BF16)
    ro, no = torch.full_like(r, 5.0), torch.full_like(r, 5.0)
    op.forward(T, x, r, ro, no, stream=stream())
    torch.cuda.synchronize()
    for v in (y, ro, no):
        assert bool((v[T:] == 5).all()) and bool(torch.isfinite(v[:T]).all())


def far_rows(T, n, dtype=BF16, value=None):
    """[T, n] rows 2^28 + 8 elements apart: from row 16 on, offsets pass 32 bits."""
    big = torch.empty((T, (1 << 28) + 8), dtype=dtype, device="cuda")
    v = big[:, :n]
    if value is not None:
        v.copy_(value)
    return v


@pytest.mark.parametrize("gs", [32, 128])
def test_linear_offsets_past_32_bits(gs):
    T = 20
    w = Weight(150, 256, gs, True, seed=41)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T, w.K), generator=gen(3), device="cuda").to(BF16)
    xf, yf = far_rows(T, w.K, value=x), far_rows(T, w.M)
    lin.forward(xf, T, yf, R=yf.copy_(torch.ones((T, w.M), device="cuda")), stream=stream())
    y = torch.empty((T, w.M), dtype=BF16, device="cuda")
    lin.forward(x, T, y, R=torch.ones_like(y), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(yf, y)
    for t in (1, 8):  # the kernel of few tokens, its rows far behind one another
        y = torch.empty((t, w.M), dtype=BF16, device="cuda")
        lin.forward(x[:t], t, y, stream=stream())
        lin.forward(xf[20 - t * 2::2] if t == 8 else xf[:1], t, yf, stream=stream())
        want = torch.empty_like(y)
        lin.forward(x[20 - t * 2::2].contiguous() if t == 8 else x[:1], t, want, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(yf[:t], want)


def test_norm_offsets_past_32_bits():
    T, H = 20, 300
    op = L.ResidualNorm(H, post="rms", pre="layer")
    b, r = (torch.randn((T, H), generator=gen(i), device="cuda").to(BF16) for i in (4, 5))
    ro, no = torch.empty_like(r), torch.empty_like(r)
    op.forward(T, b, r, ro, no, stream=stream())
    bf, rf, nf = far_rows(T, H, value=b), far_rows(T, H, value=r), far_rows(T, H)
    op.forward(T, bf, rf, rf, nf, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(rf, ro) and torch.equal(nf, no)


def test_select_offsets_past_32_bits():
    B, W, V = 4, 5, 5000
    x = torch.randn((B * W, V), generator=gen(6), device="cuda").to(BF16)
    scores = torch.randn((B, W), generator=gen(7), device="cuda")
    want = run_select(x, scores, None, -1, 6)
    got = run_select(far_rows(B * W, V, value=x), scores, None, -1, 6)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_reorder_offsets_past_32_bits():
    W, row = 4, 1200 * 1000 * 1000 + 48
    src = torch.empty((1, W, row), dtype=torch.uint8, device="cuda")
    for i in range(W):
        src[0, i] = torch.randint(0, 256, (1 << 20,), generator=gen(i), device="cuda", dtype=torch.uint8).repeat(
            row // (1 << 20) + 1)[:row]
    dst = torch.zeros_like(src)
    parent = torch.tensor([[3, 0, 3, 2]], dtype=torch.int32, device="cuda")
    L.BeamReorder([src], [dst], 1, W, W).run(parent, stream=stream())
    torch.cuda.synchronize()
    for i, p in enumerate((3, 0, 3, 2)):
        assert torch.equal(dst[0, i], src[0, p])


def test_captured_calls_with_their_own_workspaces():
    """Two captured selections, each with its own workspace, replayed in turn
    and at once on two streams."""
    B, W, V, k = 3, 6, 30011, 6
    cases = []
    for i in range(2):
        x = torch.randn((B * W, V), generator=gen(50 + i), device="cuda").to(BF16)
        scores = torch.randn((B, W), generator=gen(60 + i), device="cuda")
        want = run_select(x, scores, None, -1, k)
        bs = L.BeamSearch(B, W, V, k)
        ws = torch.empty(bs.workspace_bytes(), device="cuda", dtype=torch.uint8)
        outs = [torch.zeros((B, k), dtype=torch.int32, device="cuda"), torch.zeros((B, k), dtype=torch.int32, device="cuda"),
                torch.zeros((B, k), device="cuda"), torch.zeros((B, k), dtype=torch.uint8, device="cuda")]
        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            bs.select(x, scores, outs[0], outs[1], outs[2], ws, ws.numel(), finished_out=outs[3],
                      stream=torch.cuda.current_stream())
        cases.append((graph, want, outs, torch.cuda.Stream(), (x, scores, ws, bs)))
    for _ in range(20):
        for graph, _, _, st, _ in cases:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, want, outs, _, _ in cases:
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


@pytest.mark.parametrize("T", [5, 12, 40])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_linear_non_finite_rows_with_zeros(T, gs):
    """With zeros too, whose product with the group sums is apart: a token with
    inf or NaN changes no other token's bits and has no finite output."""
    w = Weight(200, 512, gs, True, seed=12)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T, 512), generator=gen(10), device="cuda").to(BF16)
    clean = run_linear(lin, w, x, T, F32)
    x[1, 100] = float("inf")
    x[2, 7] = -float("inf")
    x[T - 1, 3] = float("nan")
    y = run_linear(lin, w, x, T, F32)
    keep = [t for t in range(T) if t not in (1, 2, T - 1)]
    assert torch.equal(y[keep], clean[keep])
    for t, k in ((1, 100), (2, 7), (T - 1, 3)):
        assert not bool(torch.isfinite(y[t, w.w[:, k] != 0]).any())


def test_linear_status_refuses_a_captured_stream():
    w = Weight(64, 128, 32, False, seed=13)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((12, 128), generator=gen(1), device="cuda").to(BF16)
    want = run_linear(lin, w, x, 12, F32)
    y = torch.zeros_like(want)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        lin.forward(x, 12, y, stream=torch.cuda.current_stream())
        with pytest.raises(L.LlmocError, match="captured"):
            lin.status(torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    lin.status(stream())


@pytest.mark.parametrize("H", [200, 264, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 5120, 8192, 8200])
@pytest.mark.parametrize("T", [297, 1025])
@pytest.mark.parametrize("rdt", [BF16, F32])
def test_norm_many_rows(H, T, rdt):
    """Enough rows for every variant of a wide batch."""
    c = norm_config(H, "rms", "layer", BF16, seed=H)
    op = L.ResidualNorm(H, **c)
    g = gen(T + H)
    b = (torch.randn((T, H), generator=g, device="cuda") * 2 + 0.5).to(BF16)
    r = (torch.randn((T, H), generator=g, device="cuda") * 3 - 0.25).to(rdt)
    ro, no = torch.empty_like(r), torch.empty((T, H), dtype=BF16, device="cuda")
    op.forward(T, b, r, ro, no, stream=stream())
    torch.cuda.synchronize()
    wr, er, wn, en = ref_norm(b, r, None, c)
    check_rows(ro, wr, er, "residual")
    check_rows(no, wn, en, "norm")


@pytest.mark.parametrize("B,W", [(40, 8), (3, 100), (128, 8), (129, 8), (1000, 1)])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.95, 1.0])
def test_select_many_rows_some_finished(B, W, share):
    """Finished beams and beams without a score among many: the others' rows
    keep their places."""
    V, k = 1500, min(W, 5)
    g = gen(B + W)
    logits = torch.randn((B * W, V), generator=g, device="cuda")
    scores = torch.randn((B, W), generator=g, device="cuda")
    scores[torch.rand((B, W), generator=g, device="cuda") < 0.2] = float("-inf")
    scores[0, 0] = float("nan")
    fin = (torch.rand((B, W), generator=g, device="cuda") < share).to(torch.uint8)
    check_select(logits, scores, fin, 3, k)


FIRST_CALL = """
import sys
import torch
import llmoc_b200 as L
T, M, K, gs = (int(v) for v in sys.argv[1:5])
q = torch.randint(0, 256, (M, K // 2), device="cuda", dtype=torch.uint8)
s = torch.rand((M, K // gs), device="cuda").half()
torch.cuda.synchronize()
lin = L.Int4Linear.create([L.view(q, s, None, M, K, gs, L.SCHEME_AWQ_SYM, 7)], on_device=True)
x, y = torch.randn((T, K), device="cuda").to(torch.bfloat16), torch.zeros((T, M), device="cuda")
r, n = torch.randn((T, K), device="cuda").to(torch.bfloat16), torch.zeros((T, K), device="cuda", dtype=torch.bfloat16)
norm = L.ResidualNorm(K, pre="rms")
bs = L.BeamSearch(1, T, M, T)
ws = torch.empty(bs.workspace_bytes(), device="cuda", dtype=torch.uint8)
sc, pa = torch.zeros((1, T), device="cuda"), torch.zeros((1, T), device="cuda", dtype=torch.int32)
out = [pa, pa.clone(), sc.clone()]
ro = L.BeamReorder([y.view(1, T, M)], [y.clone().view(1, T, M)], 1, T, T)
st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
def step(stream):
    norm.forward(T, x, r, None, n, stream=stream)
    lin.forward(x, T, y, stream=stream)
    bs.select(y, sc, *out, ws, ws.numel(), stream=stream)
    ro.run(out[0], stream=stream)
with torch.cuda.graph(graph, stream=st):
    step(torch.cuda.current_stream())
graph.replay()
torch.cuda.synchronize()
got = [v.clone() for v in (n, y, *out, ro._keep[1][0])]
for v in (n, y, *out, ro._keep[1][0]):
    v.zero_()
step(torch.cuda.current_stream())
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (n, y, *out, ro._keep[1][0])))
lin.status(torch.cuda.current_stream())
"""


@pytest.mark.parametrize("T,M,K,gs", [(1, 512, 1024, 128), (8, 512, 4096, 32), (40, 2048, 4096, 64)])
def test_first_calls_of_a_process_are_captured(T, M, K, gs):
    """Nothing a first call sets up keeps it out of a capture."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(os.path.abspath(L.__file__)),
                                                       os.environ.get("PYTHONPATH", "")]))
    p = subprocess.run([sys.executable, "-c", FIRST_CALL, *map(str, (T, M, K, gs))], env=env, capture_output=True,
                       text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


@pytest.mark.parametrize("V", [500, 3000, 20011, 70001])
@pytest.mark.parametrize("offset", [1000.0, -1000.0, 100.0, -30000.0])
@pytest.mark.parametrize("nan", [False, True])
def test_select_with_a_common_offset(V, offset, nan):
    """A row's log-sum does not depend on where its logits lie, nor on which of
    its tiles hold a NaN (the tolerance is check_select's, which has no term in
    the logits: the reference they are summed to is one and the same number)."""
    B, W = 3, 4
    logits = torch.randn((B * W, V), generator=gen(V), device="cuda") * 3 + offset
    logits[1] = logits[0]
    if nan:
        logits[1::2, V // 3] = float("nan")
    check_select(logits, -20 * torch.rand((B, W), generator=gen(1), device="cuda"), None, -1, 5)


@pytest.mark.parametrize("V", [3000, 20011, 131072])
@pytest.mark.parametrize("keep", [0.1, 0.001])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_select_mostly_masked(V, keep, dt):
    """A mask that leaves few tokens, the same for all beams or one for each,
    with NaN in some of the masked places."""
    B, W = 4, 4
    g = gen(V)
    for rows in (1, B * W):
        logits = torch.randn((B * W, V), generator=g, device="cuda").to(dt)
        u = torch.rand((rows, V), generator=g, device="cuda")
        logits.masked_fill_(u > keep, float("-inf"))
        logits.masked_fill_(u > 0.9999, float("nan"))
        check_select(logits, -20 * torch.rand((B, W), generator=g, device="cuda"), None, -1, 6)


def test_select_mostly_masked_takes_no_longer():
    """A lane that meets masked logits only has nothing to add and no second
    look to take: such rows are read as fast as full ones (0.95 of their time;
    3.6 times it when each of their tiles was read again)."""
    B, W, V, k = 32, 8, 248320, 8
    g = gen(9)
    full = torch.randn((B * W, V), generator=g, device="cuda").to(BF16)
    few = full.masked_fill(torch.rand((1, V), generator=g, device="cuda") > 0.001, float("-inf"))
    scores = -20 * torch.rand((B, W), generator=g, device="cuda")
    bs = L.BeamSearch(B, W, V, k)
    ws = torch.empty(bs.workspace_bytes(), device="cuda", dtype=torch.uint8)
    parent = torch.empty((B, k), dtype=torch.int32, device="cuda")
    outs = (parent, parent.clone(), torch.empty((B, k), device="cuda"))
    times = {True: [], False: []}
    for rep in range(12):  # in turn, the first two to warm up
        for masked in (False, True):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            for _ in range(10):
                bs.select(few if masked else full, scores, *outs, ws, ws.numel(), stream=stream())
            b.record()
            b.synchronize()
            times[masked].append(a.elapsed_time(b))
    assert float(np.median(times[True][2:])) < 2 * float(np.median(times[False][2:]))


def test_moe_block_refuses_a_workspace_among_its_operands(oracle):
    """A workspace that an operand shares, or that wide loads could not start in,
    is refused before anything runs."""
    layer = moe_layer(oracle)
    H, T = 512, 6
    before, after = L.ResidualNorm(H, pre="rms"), L.ResidualNorm(H, pre="rms")
    n = layer.block_workspace_bytes(T)
    whole = torch.zeros((n + 16 + T * H * 2,), dtype=torch.uint8, device="cuda")
    ws = whole[:n]
    at_end = whole[n - 16:n - 16 + T * H * 2].view(BF16).view(T, H)
    at_start = whole[:T * H * 2].view(BF16).view(T, H)
    r = torch.full((T, H), 3.0, dtype=BF16, device="cuda")
    ro, no = torch.full_like(r, 5), torch.full_like(r, 7)
    for x in (at_start, at_end):
        for args, gate in (((x, ro, no), None), ((r, x, no), None), ((r, ro, x), None), ((r, ro, no), x),
                           ((r, ro, no), x[:1]), ((r, ro, no), x[:, :1])):
            with pytest.raises(L.LlmocError, match="workspace overlaps"):
                layer.forward_block(before, after, T, *args, ws, n, gate=gate, stream=stream())
    with pytest.raises(L.LlmocError, match="not aligned"):
        layer.forward_block(before, after, T, r, ro, no, whole[8:n + 8], n, stream=stream())
    torch.cuda.synchronize()
    assert bool((whole == 0).all()) and bool((r == 3).all()) and bool((ro == 5).all()) and bool((no == 7).all())
    layer.forward_block(before, after, T, r, ro, whole[n:n + T * H * 2].view(BF16).view(T, H), ws, n, stream=stream())
    torch.cuda.synchronize()
    layer.close()


@pytest.mark.parametrize("asym", [False, True])
def test_linear_create_refuses_host_memory_as_device_views(asym):
    w = Weight(32, 64, 32, asym, seed=1)
    host = [t.cpu() if t is not None else None for t in (w.q, w.s, w.z)]
    dev = [w.q, w.s, w.z]
    for i in range(3 if asym else 2):
        v = [*dev[:i], host[i], *dev[i + 1:]]
        view = L.view(*v, 32, 64, 32, L.SCHEME_GPTQ_ASYM if asym else L.SCHEME_AWQ_SYM)
        with pytest.raises(L.LlmocError, match="not in memory of device 0"):
            L.Int4Linear.create([w.view, view], on_device=True)
    L.Int4Linear.create([w.view, w.view], on_device=True).close()
    view = L.view(*host, 32, 64, 32, L.SCHEME_GPTQ_ASYM if asym else L.SCHEME_AWQ_SYM)
    L.Int4Linear.create([view], on_device=False).close()
    pinned = [t.pin_memory() if t is not None else None for t in host]  # the device can read it
    view = L.view(*pinned, 32, 64, 32, L.SCHEME_GPTQ_ASYM if asym else L.SCHEME_AWQ_SYM)
    L.Int4Linear.create([view], on_device=True).close()


@pytest.mark.parametrize("M,K,gs,T", [(20000, 6144, 128, 16), (20016, 6176, 32, 16), (20001, 6176, 64, 13),
                                      (40000, 10240, 128, 8), (64, 99968, 128, 8)])
@pytest.mark.parametrize("asym", [False, True])
def test_linear_restages_activations(M, K, gs, T, asym):
    """A CTA's share of K in more than one slab of staged activations: tile
    groups after one another in a wide matrix, a split K in a long one."""
    w = Weight(M, K, gs, asym, seed=M + K)
    lin = L.Int4Linear.create([w.view], on_device=True)
    for pad in (0, 3):
        x = torch.randn((T, K + pad), generator=gen(T), device="cuda").to(BF16)[:, :K]
        y = x.double() @ w.w.t()
        got = run_linear(lin, w, x, T, F32)
        close(got, y, w.tol(x, y, F32))
        assert torch.equal(got, run_linear(lin, w, x, T, F32))
    lin.status(stream())
    lin.close()


@pytest.mark.parametrize("M,K,gs,zp", [(300, 1408, 64, 7), (140, 992, 32, 7), (1000, 1024, 128, 7), (200, 640, 128, 20)])
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("T", [200, 512, 2049])
def test_linear_of_a_prompt(M, K, gs, zp, asym, T):
    w = Weight(M, K, gs, asym, seed=M + T, zp=zp)
    lin = L.Int4Linear.create([w.view], on_device=True)
    x = torch.randn((T, K), generator=gen(T), device="cuda").to(BF16)
    r = torch.randn((T, M), generator=gen(T + 1), device="cuda").to(BF16)
    y = x.double() @ w.w.t()
    close(run_linear(lin, w, x, T, F32), y, w.tol(x, y, F32), "fp32")
    yr = y + r.double()
    close(run_linear(lin, w, x, T, BF16, R=r), yr, w.tol(x, yr, BF16) + 2 * U * (y.abs() + r.double().abs()), "bf16")
    lin.status(stream())
    lin.close()


@pytest.mark.parametrize("V", [60, 5000, 40001])
@pytest.mark.parametrize("scale", [1e4, 1e6, 2.0 ** 24, 2.0 ** 27, 1e9, 1e15, 1e30, 1e38])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_select_with_large_logits(V, scale, dt):
    """Logits whose products with log2(e) round by far more than a bit, up to
    those whose products leave fp32, of either sign, alone or among small ones."""
    B, W, k = 3, 4, 5
    g = gen(V)
    x = torch.randn((B * W, V), generator=g, device="cuda")
    few = torch.rand((B * W, V), generator=g, device="cuda") < 0.01
    scores = -20 * torch.rand((B, W), generator=g, device="cuda")
    near = 1 + torch.round(x * 4) * 2.0 ** -23  # a few neighbours of one value
    for logits in (x * (scale / 8), -x.abs() * (scale / 8), torch.where(few, x * (scale / 8), x), near * scale,
                   -near * scale):
        check_select(logits.to(dt), scores, None, -1, k)
