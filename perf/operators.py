"""Cases, inputs, plain forms and work of three operators of the experts' feed-forward path:

* ``ffn``:  the gated block ``h = silu(x Wg) * (x Wu)`` over rows sorted by expert, forward and backward;
* ``w4``:   the experts' products on 4-bit weights with group scales, from one token to a prompt;
* ``clip``: the global norm of many gradients and the clipping that follows.

``own`` chooses between the plain forms below and the library's kernels.
"""
import math

import torch

own = False

EPS = 1e-6      # added to the norm in the clipping's quotient
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a training step's gated block: a small layer, where launches count
        dict(name="ffn small layer", op="ffn", E=8, d=1024, I=2816, T=512, k=2, routing="uniform"),
        # a layer of 8 large experts on 4096 tokens: matrix products and nothing else
        dict(name="ffn large experts", op="ffn", E=8, d=4096, I=14336, T=4096, k=2, routing="uniform"),
        # 64 small experts, top-6: short contractions of the weight gradients
        dict(name="ffn fine-grained", op="ffn", E=64, d=2048, I=1408, T=8192, k=6, routing="uniform"),
        # sizes that fill no tile, some experts without rows
        dict(name="ffn ragged", op="ffn", E=7, d=520, I=1000, T=333, k=2, routing="zipf"),
        # decode of one sequence: two experts, one row each
        dict(name="w4 one token", op="w4", proj="gate_up", E=8, d=4096, I=14336, T=1, k=2, routing="uniform", group=128, zeros=False),
        # decode of a few sequences: the down projection, long contraction, few columns
        dict(name="w4 small batch down", op="w4", proj="down", E=8, d=4096, I=14336, T=16, k=2, routing="uniform", group=128, zeros=True),
        # a decode batch on skewed experts
        dict(name="w4 decode skewed", op="w4", proj="gate_up", E=8, d=4096, I=14336, T=256, k=2, routing="zipf", group=64, zeros=False),
        # fine-grained experts at decode: 64 small matrices, a few rows each
        dict(name="w4 fine-grained", op="w4", proj="gate_up", E=64, d=2048, I=1408, T=32, k=6, routing="uniform", group=32, zeros=True),
        # a prompt of 4096 tokens through the same weights
        dict(name="w4 prompt", op="w4", proj="gate_up", E=8, d=4096, I=14336, T=4096, k=2, routing="uniform", group=128, zeros=False),
        # the gradients of one layer of large experts
        dict(name="clip large experts", op="clip", tensors=2, smallest=8 * 14336 * 4096, largest=8 * 4096 * 28672, types="bf16", clips=True),
        # many tensors from one element on, of several types, anywhere in their buckets
        dict(name="clip many", op="clip", tensors=300, smallest=1, largest=200001, types="mixed", clips=True),
        # a small layer's gradients that stay below the limit
        dict(name="clip below limit", op="clip", tensors=8, smallest=1024, largest=8 * 1024 * 5632, types="fp32", clips=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _eights(rng, lo, hi):
    """A multiple of 8, spread over the logarithm: the library's rows are whole 16-byte pieces."""
    return 8 * max(1, _log_int(rng, lo / 8, hi / 8))


def draw(rng):
    op = rng.choice(["ffn", "w4", "w4", "clip"])
    if op == "clip":
        n = _log_int(rng, 1, 400)
        largest = _log_int(rng, 64, min(9e8, 1.4e9 / n))
        return dict(op="clip", tensors=n, smallest=_log_int(rng, 1, largest), largest=largest,
                    types=rng.choice(["bf16", "fp16", "fp32", "mixed"]) if largest * n < 7e8 else "bf16", clips=rng.random() < 0.8)
    routing = rng.choice(["uniform", "uniform", "zipf"])
    while True:
        E = rng.choice([1, 2, 3, 5, 8, 8, 16, 31, 64])
        k = min(E, rng.choice([1, 2, 2, 4, 6, 8]))
        d, I = _eights(rng, 256, 6144), _eights(rng, 256, 16384)
        T = _log_int(rng, 1, 8192)
        if E * d * I <= 8 * 4096 * 14336 and T * k * d * I <= 8192 * 4096 * 14336:
            break
    c = dict(op=op, E=E, d=d, I=I, T=T, k=k, routing=routing)
    if op == "w4":
        c.update(proj=rng.choice(["gate_up", "down"]), group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------

def _preference(case):
    """How often an expert is chosen, relative to the others."""
    e = torch.arange(1, case["E"] + 1, dtype=torch.float64)
    p = e ** -1.2 if case["routing"] == "zipf" else torch.ones_like(e)
    return p / p.sum()


def _sizes(case, seed):
    """Rows per expert: every token chooses k experts, none twice."""
    g = torch.Generator().manual_seed(seed)
    chosen = torch.multinomial(_preference(case).float().expand(case["T"], -1), case["k"], replacement=False, generator=g)
    return torch.bincount(chosen.reshape(-1), minlength=case["E"])


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    """Normal values, one leading index at a time: a large tensor never exists in 32 bits."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in (out if out.dim() == 3 else [out]):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(std))
    return out


def _ceil(a, b):
    return -(-a // b)


def _tiles(codes, N, K):
    """4-bit codes of one expert ``[N, K]`` in the order the kernels read them: tiles of 16 columns by 128 k, a tile 64 lanes
    of 16 bytes, lane ``16 g + r`` with column ``r``, its word ``j`` the 8 codes of ``k = 32 j + 8 g ..``, even ones in the
    low four nibbles."""
    nt, kt = _ceil(N, 16), _ceil(K, 128)
    q = torch.zeros(nt * 16, kt * 128, dtype=torch.uint8, device=codes.device)
    q[:N, :K] = codes
    q = q.view(nt, 16, kt, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)       # [nt, kt, g, r, j, odd, i]
    q = q.reshape(nt, kt, 4, 16, 4, 4, 2)                                 # nibbles of a word in pairs: bytes
    return (q[..., 0] | (q[..., 1] << 4)).reshape(nt, kt, 1024)


def _tile_groups(v, N, groups, group):
    """Scales or zero points of one expert ``[N, groups]`` beside those tiles: ``[nt, kt, 4 column quads, groups of a tile, 4]``."""
    per = 128 // group
    nt, kt = _ceil(N, 16), _ceil(groups, per)
    s = torch.zeros(nt * 16, kt * per, dtype=v.dtype, device=v.device)
    s[:N, :groups] = v
    return s.view(nt, 4, 4, kt, per).permute(0, 3, 1, 4, 2).contiguous()


def _bucket_sizes(case):
    """Elements of each gradient, from the smallest to the largest in equal ratios."""
    n, a, b = case["tensors"], case["smallest"], case["largest"]
    return [b] if n == 1 else [int(round(a * (b / a) ** (i / (n - 1)))) for i in range(n)]


def _bucket_type(case, i):
    return TYPES[("bf16", "fp32", "bf16", "fp16")[i % 4]] if case["types"] == "mixed" else TYPES[case["types"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "clip":
        # gradients are views of one flat bucket for each type, one behind the other
        sizes = _bucket_sizes(case)
        kinds = [_bucket_type(case, i) for i in range(len(sizes))]
        flat = {t: torch.empty(sum(n for n, u in zip(sizes, kinds) if u == t), dtype=t, device="cuda") for t in dict.fromkeys(kinds)}
        for b in flat.values():
            for part in b.split(1 << 28):
                part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(0.01))
        at, grads = {t: 0 for t in flat}, []
        for n, t in zip(sizes, kinds):
            grads.append(flat[t][at[t]:at[t] + n])
            at[t] += n
        # a third of the expected norm; at most 8, so that EPS counts and a clipped bucket is clipped again by the next pass
        return {"case": case, "grads": grads, "flat": list(flat.values()),
                "max_norm": min(8.0, 0.003 * math.sqrt(sum(sizes))) if case["clips"] else 1e6}
    sizes = _sizes(case, seed)
    E, d, I, R = case["E"], case["d"], case["I"], case["T"] * case["k"]
    state = {"case": case, "sizes": sizes.cuda(), "host_sizes": sizes, "rows": sizes.tolist()}
    if case["op"] == "ffn":
        state.update(x=_randn(g, R, d), w13=_randn(g, E, d, 2 * I, std=0.02), dh=_randn(g, R, I, std=0.1))
        return state
    K, N = (d, 2 * I) if case["proj"] == "gate_up" else (I, d)
    group, groups = case["group"], _ceil(K, case["group"])
    nt, kt, per = _ceil(N, 16), _ceil(K, 128), 128 // group
    state.update(x=_randn(g, R, K), K=K, N=N,
                 codes=torch.empty(E, N, K // 2, dtype=torch.uint8, device="cuda"),
                 scales=torch.empty(E, N, groups, dtype=torch.bfloat16, device="cuda"),
                 zeros=torch.empty(E, N, groups, dtype=torch.uint8, device="cuda") if case["zeros"] else None,
                 code_tiles=torch.empty(E, nt, kt, 1024, dtype=torch.uint8, device="cuda"),
                 scale_tiles=torch.empty(E, nt, kt, 4, per, 4, dtype=torch.bfloat16, device="cuda"),
                 zero_tiles=torch.empty(E, nt, kt, 4, per, 4, dtype=torch.uint8, device="cuda") if case["zeros"] else None)
    for e in range(E):
        # what rounding a normal weight of deviation 0.02 to 16 steps gives
        q = torch.randn(N, K, generator=g, device="cuda").mul_(2.6).add_(8).round_().clamp_(0, 15).to(torch.uint8)
        s = torch.rand(N, groups, generator=g, device="cuda").mul_(0.004).add_(0.006).to(torch.bfloat16)
        state["codes"][e] = q[:, 0::2] | (q[:, 1::2] << 4)
        state["scales"][e] = s
        state["code_tiles"][e] = _tiles(q, N, K)
        state["scale_tiles"][e] = _tile_groups(s, N, groups, group)
        if case["zeros"]:
            z = torch.randint(5, 12, (N, groups), generator=g, device="cuda", dtype=torch.uint8)
            state["zeros"][e] = z
            state["zero_tiles"][e] = _tile_groups(z, N, groups, group)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"ffn": _own_ffn, "w4": _own_w4, "clip": _own_clip}[op](state)
    return {"ffn": _plain_ffn, "w4": _plain_w4, "clip": _plain_clip}[op](state)


def _own_ffn(s):
    from disagmoe_amd.grouped_gemm import ops
    x, w = s["x"].detach().requires_grad_(), s["w13"].detach().requires_grad_()
    h = ops.gmm_swiglu(x, w, s["sizes"], host_batch_sizes=s["host_sizes"])
    dx, dw = torch.autograd.grad(h, (x, w), s["dh"])
    return {"h": h.detach(), "dx": dx, "dw": dw}


def _own_w4(s):
    from disagmoe_amd.grouped_gemm import backend
    w = backend.W4Weight(s["code_tiles"], s["scale_tiles"], s["zero_tiles"], s["K"], s["N"], s["case"]["group"])
    call = backend.gmm_w4_swiglu if s["case"]["proj"] == "gate_up" else backend.gmm_w4
    return call(s["x"], w, s["sizes"], host_batch_sizes=s["host_sizes"])


def _own_clip(s):
    from disagmoe_amd.ops import grads
    norm = grads.clip_by_global_norm_(s["grads"], s["max_norm"])
    return {"norm": norm, "grads": s["flat"]}


def _by_expert(s, f, *rows):
    """f(expert, its rows of each tensor in 32 bits) of every expert."""
    parts = [t.float().split(s["rows"]) for t in rows]
    return [f(e, *p) for e, p in enumerate(zip(*parts))]


def _plain_ffn(s):
    I = s["case"]["I"]
    w = [m.float() for m in s["w13"]]
    u = torch.cat(_by_expert(s, lambda e, x: x @ w[e], s["x"]))
    gate, up = u[:, :I], u[:, I:]
    sig = torch.sigmoid(gate)
    dh = s["dh"].float()
    du = torch.cat([dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig], 1)
    dx = torch.cat(_by_expert(s, lambda e, d: d @ w[e].t(), du))
    dw = torch.stack(_by_expert(s, lambda e, x, d: (x.t() @ d).to(torch.bfloat16), s["x"], du))
    return {"h": (gate * sig * up).to(torch.bfloat16), "dx": dx.to(torch.bfloat16), "dw": dw}


def _plain_w4(s):
    def product(e, x):
        if not x.shape[0]:
            return x.new_empty(0, s["N"])
        q = s["codes"][e]
        q = torch.stack([q & 15, q >> 4], -1).view(s["N"], s["K"]).float()
        zero = 8.0 if s["zeros"] is None else spread(s["zeros"][e].float())
        return x @ ((q - zero) * spread(s["scales"][e].float())).t()

    def spread(v):
        return v.repeat_interleave(s["case"]["group"], 1)[:, :s["K"]]

    c = torch.cat(_by_expert(s, product, s["x"]))
    if s["case"]["proj"] == "gate_up":
        gate, up = c.chunk(2, 1)
        c = gate * torch.sigmoid(gate) * up
    return c.to(torch.bfloat16)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + EPS)).clamp(max=1.0)
    for g in s["grads"]:
        g.copy_(g.float() * coef)
    return {"norm": norm, "grads": s["flat"]}


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _busy(case):
    """Experts that get at least one row, on average."""
    p = (_preference(case) * case["k"]).clamp(max=1.0)
    return float((1 - (1 - p) ** case["T"]).sum())


def work(case):
    if case["op"] == "clip":
        sizes = _bucket_sizes(case)
        size = sum(n * _bucket_type(case, i).itemsize for i, n in enumerate(sizes))
        return {"bytes": (2 if case["clips"] else 1) * size + 4, "flops": (3 if case["clips"] else 2) * sum(sizes)}
    E, d, I, R = case["E"], case["d"], case["I"], case["T"] * case["k"]
    if case["op"] == "ffn":
        return {"bytes": 2 * (2 * R * d + 2 * R * I + (_busy(case) + E) * d * 2 * I) + 8 * E, "flops": 3 * 2 * R * d * 2 * I}
    K, N = (d, 2 * I) if case["proj"] == "gate_up" else (I, d)
    weight = N * K / 2 + N * _ceil(K, case["group"]) * (3 if case["zeros"] else 2)
    out = I if case["proj"] == "gate_up" else d
    return {"bytes": _busy(case) * weight + 2 * R * (K + out) + 8 * E, "flops": 2 * R * N * K}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for b in s["flat"]:
            for part in b.split(1 << 27):
                v = part.double()
                total += torch.dot(v, v)
        norm = torch.sqrt(total)
        shrink = min(1.0, s["max_norm"] / (float(norm) + EPS))
        return {"norm": norm, "grads": [b.double().mul_(shrink) for b in s["flat"]]}
    ends = torch.cumsum(s["host_sizes"], 0).tolist()
    spans = list(zip([0] + ends[:-1], ends))
    if case["op"] == "ffn":
        # gradients by differentiation of the definition
        h, dx, dw = [], [], []
        for (a, b), m in zip(spans, s["w13"]):
            x, m = s["x"][a:b].double().requires_grad_(), m.double().requires_grad_()
            y = torch.nn.functional.silu(x @ m[:, :case["I"]]) * (x @ m[:, case["I"]:])
            gx, gm = torch.autograd.grad(y, (x, m), s["dh"][a:b].double())
            h.append(y.detach()), dx.append(gx), dw.append(gm)
        return {"h": torch.cat(h), "dx": torch.cat(dx), "dw": torch.stack(dw)}
    out = []
    for e, (a, b) in enumerate(spans):
        if a == b:
            continue
        n_of, K = s["N"], s["K"]
        w = torch.empty(n_of, K, dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s["codes"][e] % 16).double()
        w[:, 1::2] = (s["codes"][e] // 16).double()
        for i in range(s["scales"].shape[2]):
            at = slice(i * case["group"], min(K, (i + 1) * case["group"]))
            w[:, at] -= 8 if s["zeros"] is None else s["zeros"][e, :, i:i + 1].double()
            w[:, at] *= s["scales"][e, :, i:i + 1].double()
        y = torch.matmul(w, s["x"][a:b].double().t()).t()
        if case["proj"] == "gate_up":
            y = torch.nn.functional.silu(y[:, :case["I"]]) * y[:, case["I"]:]
        out.append(y)
    return torch.cat(out)
