"""The operators that a decode step needs around the MoE layer, as cases to measure.

Four operators, each reached through the binding's public entry points:

* linear   dense INT4 product on device-resident weights with group scales,
           Y = X . W^T (+ R), bf16 activations (Int4Linear.forward);
* norm     the norm after a block, its gate and residual scale, the residual
           add and the norm before the next block, in one pass (ResidualNorm);
* select   one step of beam search: log-softmax over the vocabulary, the best
           continuations over all beams of a sequence (BeamSearch.select);
* reorder  the beams' states gathered by the chosen parents (BeamReorder.run).

`own` false computes the plain form in elementary torch operations.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
MAX_T = 256  # most tokens of a drawn product


def _binding():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-on-cpu_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    import llmoc_b200

    return llmoc_b200


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one token through a square projection: the launch decides
        dict(name="linear_1x4096x4096", op="linear", T=1, M=4096, K=4096, gs=128, asym=False, out="bf16", res=False),
        # a batch of 64 through an MLP projection
        dict(name="linear_64x11008x4096", op="linear", T=64, M=11008, K=4096, gs=128, asym=False, out="bf16", res=False),
        # the output head over a large vocabulary for eight sequences, fp32 logits
        dict(name="linear_head_8x248320", op="linear", T=8, M=248320, K=2048, gs=128, asym=False, out="f32", res=False),
        # odd sizes, zero points, small groups, the residual added in the product
        dict(name="linear_odd_asym_37x4101", op="linear", T=37, M=4101, K=7264, gs=32, asym=True, out="bf16", res=True),
        # one token between two blocks
        dict(name="norm_1x2048", op="norm", T=1, H=2048, post="rms", pre="rms", res="bf16", gate="none", w="bf16"),
        # a ragged batch, an odd width, layer norms, fp32 residual stream, a gate per channel
        dict(name="norm_odd_129x5001", op="norm", T=129, H=5001, post="layer", pre="layer", res="f32", gate="channel",
             w="f32"),
        # a prompt's rows, the gate one sigmoid per token
        dict(name="norm_8192x4096", op="norm", T=8192, H=4096, post="rms", pre="rms", res="bf16", gate="token",
             w="bf16"),
        # one sequence of four beams, an odd vocabulary
        dict(name="select_1x4x32003", op="select", batch=1, beams=4, vocab=32003, n_out=4, dtype="bf16", fin=False),
        # eight sequences, twice as many candidates as beams kept
        dict(name="select_8x4x131072_k8", op="select", batch=8, beams=4, vocab=131072, n_out=8, dtype="f32", fin=False),
        # a large batch over a large vocabulary, some beams finished
        dict(name="select_32x8x248320", op="select", batch=32, beams=8, vocab=248320, n_out=8, dtype="bf16", fin=True),
        # a small model's states of one sequence
        dict(name="reorder_1x4x8k", op="reorder", batch=1, beams=4, n_out=4, tensors=4, row=8192),
        # caches of 16 layers, eight sequences of eight beams
        dict(name="reorder_8x8x256k", op="reorder", batch=8, beams=8, n_out=8, tensors=32, row=262144),
    ]


def _log(rng, lo, hi):
    import math

    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "select", "reorder"])
    if op == "linear":
        asym, gs = rng.random() < 0.4, rng.choice([32, 64, 128])
        M = _log(rng, 64, 60000)
        K = 32 * _log(rng, 8, 512)
        K = min(K, 32 * max(8, (1 << 28) // (32 * M)))
        if gs > 32 and rng.random() < 0.5:
            K = max(gs, K // gs * gs)
        T = _log(rng, 1, MAX_T)
        T = max(1, min(T, 64 * 11008 * 4096 // (M * K)))
        return dict(op=op, T=T, M=M, K=K, gs=gs, asym=asym, out=rng.choice(["bf16", "bf16", "f32"]),
                    res=rng.random() < 0.4)
    if op == "norm":
        H = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            H = max(64, H // 64 * 64)
        T = max(1, min(_log(rng, 1, 8192), 8192 * 4096 // H))
        return dict(op=op, T=T, H=H, post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "rms", "layer"]),
                    res=rng.choice(["bf16", "f32"]), gate=rng.choice(["none", "token", "channel", "full"]),
                    w=rng.choice(["bf16", "f32"]))
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = _log(rng, 500, 248320)
        batch = max(1, min(_log(rng, 1, 64), 32 * 8 * 248320 // (beams * vocab)))
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, n_out=rng.randint(1, 2) * beams,
                    dtype=rng.choice(["bf16", "f32"]), fin=rng.random() < 0.5)
    batch, beams, tensors = _log(rng, 1, 16), rng.randint(2, 16), rng.randint(1, 48)
    row = _log(rng, 128, 262144)
    row = max(128, min(row, 8 * 8 * 32 * 262144 // (batch * beams * tensors)))
    if rng.random() < 0.8:
        row = row // 16 * 16
    return dict(op=op, batch=batch, beams=beams, n_out=beams, tensors=tensors, row=row)


# ------------------------------------------------------------------ prepare

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62))
    return g


def _prepare_linear(c, g):
    T, M, K, gs = c["T"], c["M"], c["K"], c["gs"]
    ng = -(-K // gs)
    # group-wise round-to-nearest quantisation of N(0, 0.02) weights, as the
    # repository's quantiser does: nibbles 0..14 around 7, or scale and offset
    q = torch.empty((M, K // 2), dtype=torch.uint8, device=DEV)
    s = torch.empty((M, ng), dtype=torch.float16, device=DEV)
    z = torch.empty((M, ng), dtype=torch.float16, device=DEV) if c["asym"] else None
    step = max(1, (1 << 27) // K)
    for m in range(0, M, step):
        w = torch.randn((min(step, M - m), ng * gs), generator=g, device=DEV) * 0.02
        w[:, K:] = 0
        w = w.view(w.shape[0], ng, gs)
        if c["asym"]:
            lo, hi = w.amin(2), w.amax(2)
            sc = ((hi - lo) / 15).clamp_min(1e-8).half()
            zo = lo.half()
            n = ((w - zo.float()[..., None]) / sc.float()[..., None]).round().clamp(0, 15)
            z[m:m + step] = zo
        else:
            sc = (w.abs().amax(2) / 7).clamp_min(1e-8).half()
            n = (w / sc.float()[..., None]).round().clamp(-7, 8) + 7
        s[m:m + step] = sc
        n = n.view(n.shape[0], -1)[:, :K].to(torch.uint8)
        q[m:m + step] = n[:, 0::2] | (n[:, 1::2] << 4)
    x = torch.randn((T, K), generator=g, device=DEV).to(torch.bfloat16)
    r = torch.randn((T, M), generator=g, device=DEV).to(torch.bfloat16) if c["res"] else None
    st = dict(q=q, s=s, z=z, x=x, r=r,
              y=torch.empty((T, M), dtype=torch.float32 if c["out"] == "f32" else torch.bfloat16, device=DEV))
    if own:
        L = _binding()
        view = L.view(q, s, z, M, K, gs, L.SCHEME_GPTQ_ASYM if c["asym"] else L.SCHEME_AWQ_SYM)
        torch.cuda.synchronize()
        st["linear"] = L.Int4Linear.create([view], device=0, on_device=True)
    return st


def _prepare_norm(c, g):
    T, H = c["T"], c["H"]
    rdt = torch.bfloat16 if c["res"] == "bf16" else torch.float32
    wdt = torch.bfloat16 if c["w"] == "bf16" else torch.float32

    def weight(mean, std):
        return (torch.randn((H,), generator=g, device=DEV) * std + mean).to(wdt)

    st = dict(block=(torch.randn((T, H), generator=g, device=DEV) * 2 + 0.3).to(torch.bfloat16),
              res=(torch.randn((T, H), generator=g, device=DEV) * 4).to(rdt),
              post_w=weight(1, 0.2), post_b=weight(0, 0.2) if c["post"] == "layer" else None,
              pre_w=weight(1, 0.2), pre_b=weight(0, 0.2) if c["pre"] == "layer" else None,
              res_out=torch.empty((T, H), dtype=rdt, device=DEV),
              norm_out=torch.empty((T, H), dtype=torch.bfloat16, device=DEV), gate=None)
    if c["gate"] != "none":
        shape = {"token": (T, 1), "channel": (1, H), "full": (T, H)}[c["gate"]]
        st["gate"] = torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)
    if own:
        L = _binding()
        st["norm"] = L.ResidualNorm(H, post=c["post"], post_weight=st["post_w"] if c["post"] != "none" else None,
                                    post_bias=st["post_b"], pre=c["pre"], pre_weight=st["pre_w"], pre_bias=st["pre_b"],
                                    gate_act="sigmoid" if c["gate"] == "token" else "none", residual_scale=1.0,
                                    block_scale=0.5, eps=1e-6)
    return st


def _prepare_select(c, g):
    B, W, V, k = c["batch"], c["beams"], c["vocab"], c["n_out"]
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    logits = (torch.randn((B * W, V), generator=g, device=DEV) * 3).to(dt)
    logits.masked_fill_(torch.rand((1, V), generator=g, device=DEV) < 0.01, float("-inf"))  # banned tokens
    scores = -30 * torch.rand((B, W), generator=g, device=DEV)
    scores[0, 1:] = float("-inf")  # a sequence at its first step: one live beam
    fin = (torch.rand((B, W), generator=g, device=DEV) < 0.2).to(torch.uint8) if c["fin"] else None
    st = dict(logits=logits, scores=scores, fin=fin, eos=V // 2,
              parent=torch.empty((B, k), dtype=torch.int32, device=DEV),
              token=torch.empty((B, k), dtype=torch.int32, device=DEV),
              out=torch.empty((B, k), dtype=torch.float32, device=DEV),
              fin_out=torch.empty((B, k), dtype=torch.uint8, device=DEV))
    if own:
        L = _binding()
        st["beam"] = L.BeamSearch(B, W, V, k, eos_token=st["eos"], device=0)
        st["ws"] = torch.empty((st["beam"].workspace_bytes(),), dtype=torch.uint8, device=DEV)
    return st


def _prepare_reorder(c, g):
    B, W, k, n, row = c["batch"], c["beams"], c["n_out"], c["tensors"], c["row"]
    src = [torch.randint(0, 256, (B, W, row), generator=g, device=DEV, dtype=torch.uint8) for _ in range(n)]
    dst = [torch.empty((B, k, row), dtype=torch.uint8, device=DEV) for _ in range(n)]
    st = dict(src=src, dst=dst, parent=torch.randint(0, W, (B, k), generator=g, device=DEV, dtype=torch.int32))
    if own:
        L = _binding()
        st["reorder"] = L.BeamReorder(src, dst, B, W, k, device=0)
    return st


def prepare(case, seed):
    g = _gen(seed)
    st = {"linear": _prepare_linear, "norm": _prepare_norm, "select": _prepare_select,
          "reorder": _prepare_reorder}[case["op"]](case, g)
    st["case"] = case
    st["stream"] = torch.cuda.current_stream()
    return st


# ---------------------------------------------------------------------- run

def _plain_linear(st):
    c = st["case"]
    n = torch.stack([st["q"] & 15, st["q"] >> 4], 2).view(c["M"], c["K"]).float()
    s = st["s"].float().repeat_interleave(c["gs"], 1)[:, :c["K"]]
    if c["asym"]:
        w = n * s + st["z"].float().repeat_interleave(c["gs"], 1)[:, :c["K"]]
    else:
        w = (n - 7) * s
    y = st["x"].float() @ w.t()
    if st["r"] is not None:
        y = y + st["r"].float()
    return y.to(st["y"].dtype)


def _plain_normed(x, kind, w, b, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + eps) * w.float()
    return x if b is None else x + b.float()


def _plain_norm(st):
    c = st["case"]
    u = _plain_normed(st["block"].float(), c["post"], st["post_w"], st["post_b"], 1e-6)
    if st["gate"] is not None:
        gate = st["gate"].float()
        u = u * (torch.sigmoid(gate) if c["gate"] == "token" else gate)
    r = st["res"].float() + 0.5 * u
    return r.to(st["res"].dtype), _plain_normed(r, c["pre"], st["pre_w"], st["pre_b"], 1e-6).to(torch.bfloat16)


def _plain_select(st):
    # 64 bits: candidates of different beams next to the border are ordered by
    # the last bits of their beams' log-sums
    c = st["case"]
    B, W, V, k = c["batch"], c["beams"], c["vocab"], c["n_out"]
    ninf = float("-inf")
    x = st["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    cand = (st["scores"].double().view(B * W, 1) + (x - lse)).view(B, W, V)
    if st["fin"] is not None:
        at_eos = torch.arange(V, device=x.device) == st["eos"]
        stay = torch.where(at_eos, st["scores"].double()[..., None], ninf)
        cand = torch.where(st["fin"].bool()[..., None], stay, cand)
    v, i = torch.sort(cand.view(B, W * V), dim=1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k]
    live = v > ninf
    parent, token = torch.where(live, i // V, -1), torch.where(live, i % V, -1)
    fin = token == st["eos"]
    if st["fin"] is not None:
        fin = fin | (live & st["fin"].bool().gather(1, parent.clamp_min(0)))
    pad = (0, k - v.shape[1])
    return (torch.nn.functional.pad(parent, pad, value=-1).int(), torch.nn.functional.pad(token, pad, value=-1).int(),
            torch.nn.functional.pad(v, pad, value=ninf).float(), torch.nn.functional.pad(fin, pad).to(torch.uint8))


def _plain_reorder(st):
    c = st["case"]
    rows = (st["parent"].long() + torch.arange(c["batch"], device=DEV)[:, None] * c["beams"]).view(-1)
    return [s.view(c["batch"] * c["beams"], c["row"])[rows].view(c["batch"], c["n_out"], c["row"]) for s in st["src"]]


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"linear": _plain_linear, "norm": _plain_norm, "select": _plain_select,
                "reorder": _plain_reorder}[op](st)
    if op == "linear":
        st["linear"].forward(st["x"], st["x"].shape[0], st["y"], R=st["r"], stream=st["stream"])
        return st["y"]
    if op == "norm":
        st["norm"].forward(st["block"].shape[0], st["block"], st["res"], st["res_out"], st["norm_out"],
                           gate=st["gate"], stream=st["stream"])
        return st["res_out"], st["norm_out"]
    if op == "select":
        st["beam"].select(st["logits"], st["scores"], st["parent"], st["token"], st["out"], st["ws"],
                          st["ws"].numel(), finished=st["fin"], finished_out=st["fin_out"], stream=st["stream"])
        return st["parent"], st["token"], st["out"], st["fin_out"]
    st["reorder"].run(st["parent"], stream=st["stream"])
    return st["dst"]


# --------------------------------------------------------------------- work

def work(case):
    c = case
    if c["op"] == "linear":
        T, M, K = c["T"], c["M"], c["K"]
        ng = -(-K // c["gs"])
        by = M * K // 2 + M * ng * 2 * (2 if c["asym"] else 1) + T * K * 2 + T * M * (4 if c["out"] == "f32" else 2)
        return {"bytes": by + (T * M * 2 if c["res"] else 0), "flops": 2 * T * M * K}
    if c["op"] == "norm":
        T, H = c["T"], c["H"]
        r = 2 if c["res"] == "bf16" else 4
        w = 2 if c["w"] == "bf16" else 4
        gate = {"none": 0, "token": 2 * T, "channel": 2 * H, "full": 2 * T * H}[c["gate"]]
        vecs = (c["post"] != "none") + (c["post"] == "layer") + 1 + (c["pre"] == "layer")
        return {"bytes": T * H * (2 + r + r + 2) + gate + vecs * H * w, "flops": 12 * T * H}
    if c["op"] == "select":
        R, V = c["batch"] * c["beams"], c["vocab"]
        by = R * V * (2 if c["dtype"] == "bf16" else 4) + R * 5 + c["batch"] * c["n_out"] * 13
        return {"bytes": by, "flops": 4 * R * V}
    W, k = c["beams"], c["n_out"]
    read = W * (1 - (1 - 1 / W) ** k)  # distinct parents of k uniform choices
    return {"bytes": c["batch"] * c["tensors"] * c["row"] * (read + k) + 4 * c["batch"] * k, "flops": 0}


# -------------------------------------------------------------------- exact

def _exact_linear(c, st):
    # group by group: s_g * sum (q - 7) x, or s_g * sum q x + z_g * sum x
    T, M, K, gs = c["T"], c["M"], c["K"], c["gs"]
    y = torch.zeros((T, M), dtype=torch.float64, device=DEV)
    x = st["x"].double()
    for i, k in enumerate(range(0, K, gs)):
        by = st["q"][:, k // 2:min(K, k + gs) // 2].long()
        xs = x[:, k:k + gs]
        dot = xs[:, 0::2] @ (by % 16).double().t() + xs[:, 1::2] @ (by // 16).double().t()
        tot = xs.sum(1, keepdim=True)
        sc = st["s"][:, i].double()
        y += dot * sc + tot * st["z"][:, i].double() if c["asym"] else (dot - 7 * tot) * sc
    return y if st["r"] is None else y + st["r"].double()


def _exact_norm(c, st):
    def stats(x, kind):
        n = x.shape[1]
        mean = x.sum(1) / n if kind == "layer" else torch.zeros(x.shape[0], dtype=x.dtype, device=x.device)
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        return mean, 1 / (var + 1e-6).sqrt()

    x = st["block"].double()
    if c["post"] != "none":
        mean, inv = stats(x, c["post"])
        x = torch.einsum("th,t,h->th", x - mean[:, None], inv, st["post_w"].double())
        x = x + st["post_b"].double() if st["post_b"] is not None else x
    if st["gate"] is not None:
        gate = st["gate"].double()
        x = x * (1 / (1 + torch.exp(-gate)) if c["gate"] == "token" else gate)
    r = st["res"].double() + x / 2
    mean, inv = stats(r, c["pre"])
    o = torch.einsum("th,t,h->th", r - mean[:, None], inv, st["pre_w"].double())
    return r, o + st["pre_b"].double() if st["pre_b"] is not None else o


def _exact_select(c, st):
    # sequence by sequence: the best of each beam by its own sort, then the best of those
    B, W, V, k = c["batch"], c["beams"], c["vocab"], c["n_out"]
    parent = torch.full((B, k), -1, dtype=torch.int32)
    token, out = parent.clone(), torch.full((B, k), float("-inf"), dtype=torch.float64)
    fout = torch.zeros((B, k), dtype=torch.uint8)
    logp = torch.log_softmax(st["logits"].double(), 1)
    few, at = torch.sort(logp, dim=1, descending=True, stable=True)
    few, at = few[:, :k].cpu().tolist(), at[:, :k].cpu().tolist()
    scores = st["scores"].double().cpu().tolist()
    fin = st["fin"].cpu().tolist() if st["fin"] is not None else [[0] * W for _ in range(B)]
    for b in range(B):
        all_ = []
        for w in range(W):
            if scores[b][w] == float("-inf"):
                continue
            if fin[b][w]:
                all_.append((-scores[b][w], w, st["eos"]))
                continue
            all_ += [(-(scores[b][w] + v), w, t) for v, t in zip(few[b * W + w], at[b * W + w]) if v > float("-inf")]
        for j, (v, w, t) in enumerate(sorted(all_)[:k]):
            parent[b, j], token[b, j], out[b, j] = w, t, -v
            fout[b, j] = 1 if fin[b][w] or t == st["eos"] else 0
    return parent, token, out, fout


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_linear(case, st)
    if op == "norm":
        return _exact_norm(case, st)
    if op == "select":
        return _exact_select(case, st)
    rows = st["parent"].cpu().tolist()
    return [torch.stack([torch.stack([s[b, p] for p in rows[b]]) for b in range(case["batch"])]) for s in st["src"]]
