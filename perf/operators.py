"""Performance cases of the 8-bit expert path and of sorting tokens by expert.

Every case goes through the entry points a user calls (`tilelang_moe_b200.kernels`).  Six kinds of work, told apart by
`case["op"]`:

  dispatch   kernels.moe_sort(ids, E), kernels.moe_permute(x, sort)    token rows copied to their experts' places
  combine    kernels.moe_unpermute(rows, sort, weights)                expert rows weighed and added up per token
  quantize   kernels.fp8_quantize(x) / fp8_quantize_blocks(w)          16 / 32 bits -> e4m3 and a scale per 128 or 128 x 128
  swiglu     kernels.fp8_silu_mul(gate, up)                            SiLU(gate) * up -> e4m3 and a scale per 128
  gemm       kernels.fp8_gemm(a, a_scale, b, b_scale)                  dense 8-bit product
  experts    kernels.fp8_grouped_gemm(a, a_scale, b, b_scale, offsets) one 8-bit product per expert's rows

Dispatch and combine with `grad` are a training step's: the result and the gradients.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
G = 128             # elements that share a scale along the inner dimension; weights: G x G
TINY = 2.0 ** -100  # the largest magnitude of a group counts as at least this


def listed():
    return [
        # a decode step of few sequences through a small layer: one short launch or two, so the call itself counts
        dict(name="dispatch_decode", op="dispatch", T=8, H=2048, E=8, k=2, dtype="bf16", load="uniform", drop=0.0, grad=False),
        # a training batch of the largest layer: eight copies of every token row, and their gradients added up
        dict(name="dispatch_train", op="dispatch", T=8192, H=7168, E=256, k=8, dtype="bf16", load="zipf", drop=0.0, grad=True),
        # a decode step through many mid-sized experts: the weighted sum of eight rows per token
        dict(name="combine_decode", op="combine", T=32, H=4096, E=128, k=8, dtype="fp16", load="uniform", drop=0.0, grad=False),
        # a training batch with a padded tail and entries dropped at an expert's capacity
        dict(name="combine_train", op="combine", T=8000, H=4096, E=64, k=8, dtype="bf16", load="zipf", drop=0.05, grad=True),
        # activations of a prefill batch in front of the experts
        dict(name="quantize_rows", op="quantize", form="rows", E=1, M=8192, K=7168, dtype="bf16"),
        # the experts of a layer laid out once when a model is loaded
        dict(name="quantize_weights", op="quantize", form="blocks", E=8, M=2048, K=7168, dtype="bf16"),
        # between the two products of a decode step: 32 tokens on 8 experts each
        dict(name="swiglu_decode", op="swiglu", M=256, I=1536, dtype="fp16", joined=False),
        # the same of a prefill batch, an odd number of rows
        dict(name="swiglu_prefill", op="swiglu", M=32769, I=2048, dtype="bf16", joined=True),
        # a single token through a projection: the weight is read once, and nothing else matters
        dict(name="gemm_token", op="gemm", M=1, N=4096, K=7168, out="bf16"),
        # a prefill batch through a projection of the largest layer: bound by the tensor cores
        dict(name="gemm_prefill", op="gemm", M=8192, N=4096, K=7168, out="bf16"),
        # a decode step: 256 rows on 128 experts, two or three each; every touched expert's weight is read once
        dict(name="experts_decode", op="experts", M=256, N=2048, K=4096, E=128, load="uniform", out="fp16"),
        # prefill on the experts of one GPU, Zipf load: ragged groups from a few rows to thousands
        dict(name="experts_prefill", op="experts", M=32768, N=2048, K=7168, E=64, load="zipf", out="bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    """A whole number in [lo, hi], spread over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "quantize", "swiglu", "gemm", "gemm", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("dispatch", "combine"):
        k = rng.choice([1, 2, 4, 6, 8])
        H = _log_int(rng, 256, 7168, rng.choice([1, 8, 64, 64]))
        T = _log_int(rng, 1, min(16384, 8192 * 7168 * 8 // (2 * k * H)))
        return dict(op=op, T=T, H=H, E=_log_int(rng, 8, 256), k=k, dtype=dtype, load=rng.choice(["uniform", "zipf"]),
                    drop=rng.choice([0.0, 0.1]), grad=rng.random() < 0.6)
    if op == "quantize":
        form = rng.choice(["rows", "blocks"])
        E = _log_int(rng, 1, 16) if form == "blocks" else 1
        K = _log_int(rng, 128, 8192, rng.choice([1, 16, 128]))
        return dict(op=op, form=form, E=E, M=_log_int(rng, 1, min(32768, (1 << 27) // (E * K))), K=K, dtype=dtype)
    if op == "swiglu":
        I = _log_int(rng, 128, 4096, rng.choice([1, 8, 128]))
        return dict(op=op, M=_log_int(rng, 1, min(65536, (1 << 27) // I)), I=I, dtype=dtype, joined=rng.random() < 0.5)
    K = _log_int(rng, 256, 8192, rng.choice([16, 128]))
    N = _log_int(rng, 256, 8192, rng.choice([1, 8, 64]))
    out = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "gemm":
        return dict(op=op, M=_log_int(rng, 1, min(16384, (1 << 38) // (N * K))), N=N, K=K, out=out)
    E = _log_int(rng, 2, min(256, (1 << 30) // (N * K)))
    return dict(op=op, M=_log_int(rng, 1, min(32768, (1 << 38) // (N * K))), N=N, K=K, E=E, load=rng.choice(["uniform", "zipf"]), out=out)


# ------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _expert_ids(T, k, E, load, drop, g):
    """k different experts per token (fewer experts than k: with repeats); dropped entries are -1, and so are all of the
    last tokens, a padded tail, where anything is dropped."""
    pop = torch.ones(E, device="cuda") if load == "uniform" else 1.0 / torch.arange(1, E + 1, device="cuda").float() ** 1.1
    noise = -torch.log(-torch.log(torch.rand(T, E, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)))
    ids = (pop.log() + noise).topk(min(k, E), dim=1).indices
    ids = ids.repeat(1, -(-k // E))[:, :k].contiguous()
    if drop:
        ids[torch.rand(T, k, device="cuda", generator=g) < drop] = -1
        ids[T - T // 16:] = -1
    return ids.to(torch.int32)


def _sorted_tables(ids, E):
    """offsets [E + 1], perm [n] and row_of [n] of the entries sorted by expert, dropped ones behind all of them."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), E, flat)
    perm = torch.argsort(key, stable=True)
    counts = (key.unsqueeze(0) == torch.arange(E, device=key.device).unsqueeze(1)).sum(1) if key.numel() * E < 1 << 24 \
        else torch.bincount(key, minlength=E + 1)[:E]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    row_of = torch.empty_like(perm)
    row_of[perm] = torch.arange(perm.numel(), device=perm.device)
    return offsets.to(torch.int32), perm.to(torch.int32), row_of.to(torch.int32)


def _group_offsets(M, E, load, g):
    """Rows of each expert's group: M rows, each on one of E experts."""
    pop = torch.ones(E, device="cuda") if load == "uniform" else 1.0 / torch.arange(1, E + 1, device="cuda").float() ** 1.1
    picks = torch.multinomial(pop, M, replacement=True, generator=g)
    return torch.cat([picks.new_zeros(1), torch.bincount(picks, minlength=E).cumsum(0)]).to(torch.int32)


def _groups(x, rows, cols):
    """x [..., M, K] padded with zeros to whole groups: [..., M / rows, rows, K / cols, cols]."""
    M, K = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -K % cols, 0, -M % rows))
    return x.reshape(*x.shape[:-2], x.shape[-2] // rows, rows, x.shape[-1] // cols, cols)


def _quantized(x, rows):
    """e4m3 values of x and a scale per `rows` x 128: the largest magnitude of a group becomes 448."""
    M, K = x.shape[-2:]
    v = _groups(x.float(), rows, G)
    top = v.abs().amax(dim=(-3, -1), keepdim=True).clamp(min=TINY)
    q = (v * (448.0 / top)).to(E4M3)
    q = q.reshape(*v.shape[:-4], v.shape[-4] * rows, v.shape[-2] * G)[..., :M, :K].contiguous()
    return q, (top / 448.0).reshape(*v.shape[:-4], v.shape[-4], v.shape[-2])


def _activations(M, K, g, dtype=torch.float32):
    """Rows of differing size with a few large channels, as behind a normalisation."""
    x = torch.randn(M, K, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(M, 1, device="cuda", generator=g))
    x[:, :: max(1, K // 8)] *= 8.0
    return x.to(dtype)


def _weights(E, N, K, g):
    """Expert weights in 8 bits, one expert at a time: the 16-bit ones are never held together."""
    q = torch.empty(E, N, K, device="cuda", dtype=E4M3)
    s = torch.empty(E, -(-N // G), -(-K // G), device="cuda")
    for e in range(E):
        q[e], s[e] = _quantized(torch.randn(N, K, device="cuda", generator=g) / math.sqrt(K), G)
    return q, s


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    op = case["op"]
    if op in ("dispatch", "combine"):
        T, H, E, k = case["T"], case["H"], case["E"], case["k"]
        dt = DTYPES[case["dtype"]]
        s["ids"] = _expert_ids(T, k, E, case["load"], case["drop"], g)
        if op == "dispatch":
            s["x"] = torch.randn(T, H, device="cuda", generator=g).to(dt).requires_grad_(case["grad"])
            s["g"] = torch.randn(T * k, H, device="cuda", generator=g).to(dt) if case["grad"] else None
        else:
            s["offsets"], s["perm"], s["row_of"] = _sorted_tables(s["ids"], E)
            s["rows"] = torch.randn(T * k, H, device="cuda", generator=g).to(dt).requires_grad_(case["grad"])
            s["w"] = torch.softmax(torch.randn(T, k, device="cuda", generator=g), dim=1).requires_grad_(case["grad"])
            s["g"] = torch.randn(T, H, device="cuda", generator=g).to(dt) if case["grad"] else None
    elif op == "quantize":
        if case["form"] == "rows":
            s["x"] = _activations(case["M"], case["K"], g, DTYPES[case["dtype"]])
        else:
            s["x"] = (torch.randn(case["E"], case["M"], case["K"], device="cuda", generator=g) / math.sqrt(case["K"])).to(DTYPES[case["dtype"]])
    elif op == "swiglu":
        M, I, dt = case["M"], case["I"], DTYPES[case["dtype"]]
        if case["joined"]:      # both halves in the rows of one product's output
            h = (1.5 * torch.randn(M, 2 * I, device="cuda", generator=g)).to(dt)
            s["gate"], s["up"] = h[:, :I], h[:, I:]
        else:
            s["gate"], s["up"] = ((1.5 * torch.randn(M, I, device="cuda", generator=g)).to(dt) for _ in range(2))
    else:
        s["a"], s["sa"] = _quantized(_activations(case["M"], case["K"], g), 1)
        if op == "gemm":
            b, sb = _weights(1, case["N"], case["K"], g)
            s["b"], s["sb"] = b[0], sb[0]
        else:
            s["b"], s["sb"] = _weights(case["E"], case["N"], case["K"], g)
            s["offsets"] = _group_offsets(case["M"], case["E"], case["load"], g)
            s["bounds"] = s["offsets"].tolist()      # the host's copy: the plain form slices by it
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_dispatch(s):
    T, k = s["ids"].shape
    offsets, perm, row_of = _sorted_tables(s["ids"], s["E"])
    live = torch.arange(T * k, device="cuda") < offsets[-1]
    rows = torch.where(live.unsqueeze(1), s["x"].detach()[perm.long() // k], 0)
    got = {"rows": rows, "offsets": offsets, "row_of": row_of}
    if s["grad"]:
        g = torch.where(live.unsqueeze(1), s["g"], 0)[row_of.long()].view(T, k, -1)
        got["grad_x"] = g.float().sum(1).to(g.dtype)
    return got


def _plain_combine(s):
    T, k = s["ids"].shape
    at, rows, w = s["row_of"].long().view(T, k), s["rows"].detach(), s["w"].detach()
    live = at < s["offsets"][-1]
    mine = torch.where(live.unsqueeze(2), rows[at], 0).float()
    got = {"y": (w.unsqueeze(2) * mine).sum(1).to(rows.dtype)}
    if s["grad"]:
        gy = s["g"].float().unsqueeze(1)
        got["grad_rows"] = torch.zeros_like(rows)
        got["grad_rows"][at] = torch.where(live.unsqueeze(2), w.unsqueeze(2) * gy, 0.0).to(rows.dtype)
        got["grad_w"] = (mine * gy).sum(2)
    return got


def _dequantized(q, scale, rows):
    """The fp32 values that 8-bit ones and their scales stand for."""
    M, K = q.shape
    v = _groups(q.float(), rows, G) * scale.unsqueeze(1).unsqueeze(3)
    return v.reshape(-1, v.shape[-2] * G)[:M, :K]


def _plain_gemm(s):
    y = _dequantized(s["a"], s["sa"], 1) @ _dequantized(s["b"], s["sb"], G).T
    return y.to(DTYPES[s["out"]])


def _plain_experts(s):
    a = _dequantized(s["a"], s["sa"], 1)
    at = s["bounds"]
    return torch.cat([(a[at[e]:at[e + 1]] @ _dequantized(s["b"][e], s["sb"][e], G).T).to(DTYPES[s["out"]])
                      for e in range(s["E"])])


def run(state):
    s, op = state, state["op"]
    if own:
        from tilelang_moe_b200 import kernels
        if op == "dispatch":
            sort = kernels.moe_sort(s["ids"], s["E"])
            rows = kernels.moe_permute(s["x"], sort)
            got = {"rows": rows.detach(), "offsets": sort.offsets, "row_of": sort.row_of}
            if s["grad"]:
                got["grad_x"], = torch.autograd.grad(rows, s["x"], s["g"])
            return got
        if op == "combine":
            sort = kernels.MoESort(s["offsets"], s["perm"], s["row_of"], s["k"])
            y = kernels.moe_unpermute(s["rows"], sort, s["w"])
            got = {"y": y.detach()}
            if s["grad"]:
                got["grad_rows"], got["grad_w"] = torch.autograd.grad(y, (s["rows"], s["w"]), s["g"])
            return got
        if op == "quantize":
            q, scale = kernels.fp8_quantize(s["x"]) if s["form"] == "rows" else kernels.fp8_quantize_blocks(s["x"])
            return {"q": q, "scale": scale}
        if op == "swiglu":
            q, scale = kernels.fp8_silu_mul(s["gate"], s["up"])
            return {"q": q, "scale": scale}
        if op == "gemm":
            return {"y": kernels.fp8_gemm(s["a"], s["sa"], s["b"], s["sb"], out_dtype=DTYPES[s["out"]])}
        return {"y": kernels.fp8_grouped_gemm(s["a"], s["sa"], s["b"], s["sb"], s["offsets"], out_dtype=DTYPES[s["out"]])}
    if op == "dispatch":
        return _plain_dispatch(s)
    if op == "combine":
        return _plain_combine(s)
    if op == "quantize":
        q, scale = _quantized(s["x"], 1 if s["form"] == "rows" else G)
        return {"q": q, "scale": scale}
    if op == "swiglu":
        gate, up = s["gate"].float(), s["up"].float()
        q, scale = _quantized(gate / (1 + torch.exp(-gate)) * up, 1)
        return {"q": q, "scale": scale}
    return {"y": _plain_gemm(s) if op == "gemm" else _plain_experts(s)}


# ------------------------------------------------------------------------------------------------------- work, exact
def work(case):
    op = case["op"]
    if op in ("dispatch", "combine"):
        T, H, k, w = case["T"], case["H"], case["k"], 4 if case["dtype"] == "fp32" else 2
        one, many = T * H * w, T * k * H * w
        tables = 4 * T * k
        if op == "dispatch":        # ids read, row_of and offsets written; with gradients the reverse copy
            moved = one + many + 2 * tables + 4 * (case["E"] + 1) + (one + many if case["grad"] else 0)
            return {"bytes": moved, "flops": T * k * H if case["grad"] else 0}
        # rows and the incoming gradient are read once each, their gradients written
        moved = one + many + 2 * tables + (one + many + tables if case["grad"] else 0)
        return {"bytes": moved, "flops": (5 if case["grad"] else 2) * T * k * H}
    if op == "quantize":
        n, w = case["E"] * case["M"] * case["K"], 4 if case["dtype"] == "fp32" else 2
        rows = case["M"] if case["form"] == "rows" else -(-case["M"] // G)
        return {"bytes": n * (w + 1) + 4 * case["E"] * rows * -(-case["K"] // G), "flops": 2 * n}
    if op == "swiglu":
        n, w = case["M"] * case["I"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * (2 * w + 1) + 4 * case["M"] * -(-case["I"] // G), "flops": 7 * n}
    M, N, K, w = case["M"], case["N"], case["K"], 4 if case["out"] == "fp32" else 2
    E = 1
    if op == "experts":             # experts that M draws are expected to touch
        pop = [1.0 if case["load"] == "uniform" else (e + 1) ** -1.1 for e in range(case["E"])]
        total = sum(pop)
        E = sum(1 - (1 - p / total) ** M for p in pop)
    groups = -(-K // G)
    return {"bytes": M * K + 4 * M * groups + E * (N * K + 4 * -(-N // G) * groups) + M * N * w, "flops": 2 * M * N * K}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("dispatch", "combine"):
        ids = s["ids"].reshape(-1).cpu().tolist()
        T, k, E = case["T"], case["k"], case["E"]
        if T * k > 1 << 20:
            return None
        buckets = [[] for _ in range(E + 1)]
        for i, e in enumerate(ids):
            buckets[e if 0 <= e < E else E].append(i)
        order = [i for b in buckets for i in b]
        kept = len(order) - len(buckets[E])
        perm = torch.tensor(order, device="cuda")
        token = perm[:kept] // k
        if op == "dispatch":
            x = s["x"].detach().double()
            got = {"rows": torch.zeros(T * k, case["H"], device="cuda", dtype=torch.float64), "offsets": None, "row_of": None}
            got["rows"][:kept] = x[token]
            if case["grad"]:
                got["grad_x"] = torch.zeros_like(x).index_add_(0, token, s["g"][:kept].double())
            return got
        w, rows = s["w"].detach().double().reshape(-1)[perm[:kept]], s["rows"].detach()
        y = torch.zeros(T, case["H"], device="cuda", dtype=torch.float64)
        got = {"y": y.index_add_(0, token, rows[:kept].double() * w.unsqueeze(1))}
        if case["grad"]:
            gy = s["g"].double()[token]
            got["grad_rows"] = torch.zeros(rows.shape, device="cuda", dtype=torch.float64)
            got["grad_rows"][:kept] = gy * w.unsqueeze(1)
            got["grad_w"] = torch.zeros(T * k, device="cuda", dtype=torch.float64)
            got["grad_w"][perm[:kept]] = torch.linalg.vecdot(gy, rows[:kept].double())
            got["grad_w"] = got["grad_w"].view(T, k)
        return got
    if op in ("quantize", "swiglu"):
        if op == "swiglu":
            gate, up = s["gate"].double(), s["up"].double()
            x = gate * torch.sigmoid(gate) * up
        else:
            x = s["x"].double()
        x = x.reshape(-1, *x.shape[-2:])
        rows = G if case.get("form") == "blocks" else 1
        # the largest magnitude along each group of 128, then over the rows that share a scale
        ends = torch.arange(x.shape[2], device="cuda") // G
        top = torch.zeros(*x.shape[:2], int(ends[-1]) + 1, device="cuda", dtype=torch.float64)
        top.scatter_reduce_(2, ends.expand(*x.shape[:2], -1).contiguous(), x.abs(), "amax")
        if rows > 1:
            top = torch.stack([part.amax(1) for part in top.split(rows, dim=1)], 1)
        top = top.clamp(min=TINY)
        # no 64-bit value stands for the 8-bit one: it is the nearest of a grid, here the value on that grid
        return {"q": None, "scale": (top / 448.0).reshape(s["x"].shape[:-2] + top.shape[1:] if op == "quantize" else top.shape[1:])}
    a, sa = s["a"].double(), s["sa"].double()
    if op == "gemm":
        y = _exact_product(a, sa, s["b"], s["sb"])
        return {"y": y}
    y = torch.empty(case["M"], case["N"], device="cuda", dtype=torch.float64)
    at = s["bounds"]
    for e in range(case["E"]):
        if at[e + 1] > at[e]:
            y[at[e]:at[e + 1]] = _exact_product(a[at[e]:at[e + 1]], sa[at[e]:at[e + 1]], s["b"][e], s["sb"][e])
    return {"y": y}


def _exact_product(a, sa, b, sb):
    """One block of 128 along the inner dimension at a time, each with its scales."""
    N, K = b.shape
    of_row = torch.arange(N, device="cuda") // G
    y = torch.zeros(a.shape[0], N, device="cuda", dtype=torch.float64)
    for i in range(-(-K // G)):
        part = a[:, i * G:(i + 1) * G] @ b[:, i * G:(i + 1) * G].double().T
        y += part * sa[:, i:i + 1] * sb.double()[of_row, i]
    return y
