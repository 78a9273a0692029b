"""Speed and exactness of the operators of pretraining on packed documents.

Three operators that one training step of the BERT path calls together:

* the embedding lookup: a sum of scaled rows of one to three tables (tokens,
  positions, segments), with the tables' gradients;
* attention inside documents that lie one behind the other in one batch of
  tokens, with scores that may fall off with distance, and its gradients;
* the Newton-Schulz orthogonalisation of a momentum, by which the Muon
  optimiser turns it into an update.

``own`` chooses between their plain form (elementary torch operations in 32
bits, rounded once at the end) and this package's entry points.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# Newton-Schulz: X <- a X + (b A + c A A) X with A = X X^T
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_EPS = 1e-7


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one short sequence that is scored, not trained: latency
        {"name": "embed eval 128", "op": "embed", "tokens": 128, "hidden": 768,
         "vocab": 30528, "tables": 3, "dtype": "bf16", "train": False},
        # BERT-base, 32 sequences of 512: the three tables and their gradients
        {"name": "embed train 16384", "op": "embed", "tokens": 16384,
         "hidden": 768, "vocab": 30528, "tables": 3, "dtype": "bf16",
         "train": True},
        # BERT-large's width, a large batch, the token table alone
        {"name": "embed train 65536", "op": "embed", "tokens": 65536,
         "hidden": 1024, "vocab": 30528, "tables": 1, "dtype": "bf16",
         "train": True},
        # odd sizes in full precision (a small vocabulary, an odd width)
        {"name": "embed train odd fp32", "op": "embed", "tokens": 3001,
         "hidden": 201, "vocab": 1009, "tables": 2, "dtype": "fp32",
         "train": True},
        # one short document that is scored: latency
        {"name": "attn eval 128", "op": "attn", "tokens": 128, "longest": 128,
         "ragged": False, "heads": 12, "kv_heads": 12, "dim": 64,
         "dtype": "bf16", "slopes": False, "train": False},
        # BERT-base's phase of short sequences: 32 of 128 tokens
        {"name": "attn train 32x128", "op": "attn", "tokens": 4096,
         "longest": 128, "ragged": False, "heads": 12, "kv_heads": 12,
         "dim": 64, "dtype": "bf16", "slopes": False, "train": True},
        # documents of 1 to 512 tokens packed into 32 rows of 512, padding
        # behind the last one, scores that fall off with distance
        {"name": "attn train packed 16384", "op": "attn", "tokens": 16384,
         "longest": 512, "ragged": True, "heads": 12, "kv_heads": 12,
         "dim": 64, "dtype": "bf16", "slopes": True, "train": True},
        # long documents, wide heads, four query heads on each key head
        {"name": "attn train long grouped", "op": "attn", "tokens": 8192,
         "longest": 4096, "ragged": True, "heads": 16, "kv_heads": 4,
         "dim": 128, "dtype": "fp16", "slopes": False, "train": True},
        # two very long documents that are scored
        {"name": "attn eval 2x8192", "op": "attn", "tokens": 16384,
         "longest": 8192, "ragged": False, "heads": 12, "kv_heads": 12,
         "dim": 64, "dtype": "bf16", "slopes": True, "train": False},
        # one small matrix: latency
        {"name": "muon 64x128", "op": "muon", "batch": 1, "rows": 64,
         "cols": 128},
        # BERT-base's attention projections, all layers at once
        {"name": "muon 12x2304x768", "op": "muon", "batch": 12, "rows": 2304,
         "cols": 768},
        # BERT-large's feed-forward matrices, all layers at once
        {"name": "muon 24x1024x4096", "op": "muon", "batch": 24, "rows": 1024,
         "cols": 4096},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("embed", "attn", "muon"))
    if op == "embed":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        hidden = rng.choice((rng.randint(1, 300), 8 * rng.randint(1, 128)))
        return {"op": op, "tokens": _log(rng, 1, 60000), "hidden": hidden,
                "vocab": _log(rng, 2, 60000), "tables": rng.randint(1, 3),
                "dtype": dtype, "train": rng.random() < 0.7}
    if op == "attn":
        group = rng.choice((1, 1, 1, 2, 4))
        kv_heads = rng.randint(1, 16 // group)
        longest = _log(rng, 1, 2048)
        tokens = min(16384, longest * _log(rng, 1, 64) + rng.randint(0, 40))
        return {"op": op, "tokens": max(tokens, longest), "longest": longest,
                "ragged": rng.random() < 0.7, "heads": group * kv_heads,
                "kv_heads": kv_heads, "dim": 8 * rng.randint(2, 16),
                "dtype": rng.choice(("bf16", "bf16", "fp16")),
                "slopes": rng.random() < 0.5, "train": rng.random() < 0.6}
    return {"op": op, "batch": _log(rng, 1, 12), "rows": _log(rng, 1, 2400),
            "cols": _log(rng, 1, 2400)}


def _lengths(case):
    """The documents' lengths: the same for every seed, in another order."""
    tokens, longest = case["tokens"], case["longest"]
    if not case["ragged"]:
        return [longest] * (tokens // longest)
    rng = random.Random(tokens * 8209 + longest)
    room = tokens - tokens // 64          # what is left is padding
    got = [longest] if longest <= room else []
    room -= sum(got)
    while room > 0:
        n = int(longest * rng.lognormvariate(-0.8, 0.7))
        n = max(1, min(n, longest, room))
        got.append(n)
        room -= n
    if len(got) > 2:
        got.append(0)                     # an unused slot of a fixed-size batch
    return got


def _embed_sizes(case):
    """Rows of each table."""
    return [case["vocab"], 512, 2][:case["tables"]]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _embed_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, h, t = case["tokens"], case["hidden"], DTYPES[case["dtype"]]
    sizes = _embed_sizes(case)
    # tokens as text has them: a word's rank by a power law, and one token in
    # eight masked; positions that restart; two segments
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(sizes[0] + 1.0)).long() - 1)
    ids = ids.clamp_(0, sizes[0] - 1)
    ids[torch.rand(n, generator=g, device="cuda") < 0.12] = sizes[0] // 3
    first = int(torch.randint(0, 512, (1,), generator=g, device="cuda"))
    place = (torch.arange(n, device="cuda") + first) % 512
    segment = (place >= 200).long()
    tables = [torch.randn(v, h, generator=g, device="cuda").mul_(0.02).to(t)
              for v in sizes]
    grad = torch.randn(n, h, generator=g, device="cuda").to(t)
    scales = [math.sqrt(h), 1.0, 1.0][:len(sizes)]
    return {"ids": [ids, place, segment][:len(sizes)], "tables": tables,
            "scales": scales, "grad": grad}


def _attn_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    n, h, kh, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    ends = [0]
    for x in lengths:
        ends.append(ends[-1] + x)
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    new = {"cu": cu, "scale": d ** -0.5, "slopes": None,
           "grad": torch.randn(n, h, d, generator=g, device="cuda").to(t)}
    if case["slopes"]:
        new["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h)
                                      for i in range(h)], device="cuda")
    if kh == h:                           # one projection's output
        new["qkv"] = torch.randn(n, 3, h, d, generator=g, device="cuda").to(t)
    else:
        for name, heads in (("q", h), ("k", kh), ("v", kh)):
            new[name] = torch.randn(n, heads, d, generator=g,
                                    device="cuda").to(t)
    return new


def _muon_inputs(case, seed):
    # a momentum: a few strong directions, a long tail, some noise
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, n, m = case["batch"], case["rows"], case["cols"]
    r = min(n, m)
    s = torch.arange(1, r + 1, device="cuda").float().rsqrt()
    left = torch.randn(b, n, r, generator=g, device="cuda") * s
    right = torch.randn(b, r, m, generator=g, device="cuda")
    noise = torch.randn(b, n, m, generator=g, device="cuda")
    return {"g": (left @ right + 0.3 * noise) * 1e-3}


def prepare(case, seed):
    make = {"embed": _embed_inputs, "attn": _attn_inputs, "muon": _muon_inputs}
    state = make[case["op"]](case, seed)
    if case.get("train"):
        for name in ("tables", "qkv", "q", "k", "v"):
            leaves = state.get(name, ())
            for x in leaves if isinstance(leaves, list) else [leaves]:
                if isinstance(x, torch.Tensor):
                    x.requires_grad_(True)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _plain_embed(s):
    ids, tables, scales, grad = s["ids"], s["tables"], s["scales"], s["grad"]
    t = tables[0].dtype
    rows = [w.detach().float()[i] * c for i, w, c in zip(ids, tables, scales)]
    out = {"out": sum(rows[1:], rows[0]).to(t)}
    if s["case"]["train"]:
        out["grads"] = [
            torch.zeros(w.shape, dtype=torch.float32, device=w.device)
            .index_add_(0, i, grad.float() * c).to(t)
            for i, w, c in zip(ids, tables, scales)]
    return out


def _padded(x, index):
    """[T, H, D] tokens -> [documents, H, L, D] in 32 bits."""
    return x.detach().float()[index].transpose(1, 2).contiguous()


def _plain_attn(s):
    case, cu, scale = s["case"], s["cu"].long(), s["scale"]
    n, longest = case["tokens"], case["longest"]
    group = case["heads"] // case["kv_heads"]
    q, k, v = s["qkv"].unbind(1) if "qkv" in s else (s["q"], s["k"], s["v"])
    t, dev = q.dtype, q.device
    place = torch.arange(longest, device=dev)
    inside = place < (cu[1:] - cu[:-1])[:, None]           # [documents, L]
    index = torch.where(inside, cu[:-1, None] + place, 0)
    token = torch.arange(n, device=dev)
    doc = (token[:, None] >= cu[1:]).sum(1)                # of each token
    real = (doc < len(cu) - 1)[:, None, None]
    doc = doc.clamp(max=len(cu) - 2)
    at = (token - cu[doc]).clamp(0, longest - 1)

    def back(x):                                           # to [T, H, D]
        return torch.where(real, x.transpose(1, 2)[doc, at], 0.0).to(t)

    keep = (inside[:, None, :, None] & inside[:, None, None, :])
    qp = _padded(q, index)
    kp = _padded(k, index).repeat_interleave(group, 1)
    vp = _padded(v, index).repeat_interleave(group, 1)
    x = qp @ kp.transpose(2, 3).contiguous()
    x *= scale
    if s["slopes"] is not None:
        far = (place[:, None] - place).abs().float()
        x -= s["slopes"][:, None, None] * far
    x = torch.where(keep, x, -torch.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -torch.inf, 0.0, top))
    p = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    out = {"out": back(p @ vp)}
    if not case["train"]:
        return out
    gp = torch.where(inside[:, None, :, None], _padded(s["grad"], index), 0.0)
    dv = p.transpose(2, 3).contiguous() @ gp
    dp = gp @ vp.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = ds @ kp
    dk = ds.transpose(2, 3).contiguous() @ qp
    if group > 1:
        dk, dv = (y.unflatten(1, (-1, group)).sum(2) for y in (dk, dv))
    if "qkv" in s:
        out["dqkv"] = torch.stack([back(dq), back(dk), back(dv)], 1)
    else:
        out.update(dq=back(dq), dk=back(dk), dv=back(dv))
    return out


def _plain_step(x):
    a = x @ x.transpose(1, 2).contiguous()
    return NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x


def _plain_muon(s):
    g = s["g"]
    tall = g.shape[1] > g.shape[2]
    x = (g.transpose(1, 2) if tall else g).contiguous()
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt() + NS_EPS
    x = x / norm.float()
    x = _plain_step(_plain_step(_plain_step(_plain_step(_plain_step(x)))))
    x = x.transpose(1, 2) if tall else x
    return {"out": x.to(torch.bfloat16).contiguous()}


# ---------------------------------------------------------------------------
# this package's operators
# ---------------------------------------------------------------------------

def _own_embed(s):
    from deeplearning_cfn_amd.ops import functional as F_amd
    y = F_amd.embedding_sum(s["ids"], s["tables"], s["scales"])
    out = {"out": y.detach()}
    if s["case"]["train"]:
        out["grads"] = list(torch.autograd.grad(y, s["tables"], s["grad"]))
    return out


def _own_attn(s):
    from deeplearning_cfn_amd.ops import functional as F_amd
    if "qkv" in s:
        y = F_amd.document_attention_qkv(s["qkv"], s["cu"], scale=s["scale"],
                                         slopes=s["slopes"])
    else:
        y = F_amd.document_attention(s["q"], s["k"], s["v"], s["cu"],
                                     scale=s["scale"], slopes=s["slopes"])
    out = {"out": y.detach()}
    if s["case"]["train"]:
        if "qkv" in s:
            out["dqkv"], = torch.autograd.grad(y, [s["qkv"]], s["grad"])
        else:
            out["dq"], out["dk"], out["dv"] = torch.autograd.grad(
                y, [s["q"], s["k"], s["v"]], s["grad"])
    return out


def _own_muon(s):
    from deeplearning_cfn_amd.ops import functional as F_amd
    return {"out": F_amd.newton_schulz(s["g"], steps=5, eps=NS_EPS)}


def run(state):
    if own:
        form = {"embed": _own_embed, "attn": _own_attn, "muon": _own_muon}
    else:
        form = {"embed": _plain_embed, "attn": _plain_attn,
                "muon": _plain_muon}
    return form[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "embed":
        n, h, e = case["tokens"], case["hidden"], BYTES[case["dtype"]]
        sizes = _embed_sizes(case)
        rows = sum(min(n, v) for v in sizes)
        total = len(sizes) * n * 8 + (rows + n) * h * e
        flops = 2 * len(sizes) * n * h
        if case["train"]:
            total += (n + sum(sizes)) * h * e
            flops *= 2
        return {"bytes": total, "flops": flops}
    if case["op"] == "attn":
        n, h, kh, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        square = sum(x * x for x in _lengths(case))
        q, kv = n * h * d * 2, n * kh * d * 2
        total, flops = 2 * q + 2 * kv, 4 * square * h * d
        if case["train"]:                 # the gradient in, three out
            total += 2 * q + 2 * kv
            flops += 10 * square * h * d
        return {"bytes": total, "flops": flops}
    b = case["batch"]
    n, m = sorted((case["rows"], case["cols"]))
    # X X^T and A A are symmetric: half of each product
    step = n * n * m + n * n * n + 2 * n * n * m
    return {"bytes": b * n * m * (4 + 2),
            "flops": 5 * b * step}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_embed(case, s):
    n, tables = case["tokens"], s["tables"]
    y = torch.zeros(n, case["hidden"], dtype=torch.float64, device="cuda")
    grads = []
    for i, w, c in zip(s["ids"], tables, s["scales"]):
        y += torch.index_select(w.detach().double(), 0, i) * c
        d = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        order = torch.argsort(i, stable=True)
        # running sums over the sorted tokens, differences at the rows' ends
        run_ = torch.cumsum(s["grad"].double()[order], 0)
        ends = torch.bincount(i, minlength=w.shape[0]).cumsum(0)
        upto = torch.cat([torch.zeros_like(run_[:1]), run_])[ends]
        d[0] = upto[0]
        d[1:] = upto[1:] - upto[:-1]
        grads.append(d * c)
    return {"out": y, "grads": grads} if case["train"] else {"out": y}


def _exact_attn(case, s):
    names = ["qkv"] if "qkv" in s else ["q", "k", "v"]
    whole = [s[x].detach() for x in names]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["grad"].shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x.shape, dtype=torch.float64, device="cuda")
             for x in whole]
    ends = s["cu"].tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        if a == b:
            continue
        mine = [x[a:b].double().requires_grad_(case["train"]) for x in whole]
        q, k, v = mine[0].unbind(1) if len(mine) == 1 else mine
        k, v = (x[:, torch.arange(case["heads"], device="cuda") // group]
                for x in (k, v))
        x = torch.bmm(q.transpose(0, 1).contiguous(),
                      k.permute(1, 2, 0).contiguous()) * s["scale"]
        if s["slopes"] is not None:
            at = torch.arange(b - a, device="cuda").double()
            x = x - (s["slopes"].double()[:, None, None]
                     * torch.abs(at[None, :] - at[:, None]))
        w = torch.exp(x - torch.logsumexp(x, 2, keepdim=True))
        y = torch.bmm(w, v.transpose(0, 1).contiguous()).transpose(0, 1)
        out[a:b] = y.detach()
        if case["train"]:
            got = torch.autograd.grad(y, mine, s["grad"][a:b].double())
            for g, d in zip(grads, got):
                g[a:b] = d
        del x, w, y
    if not case["train"]:
        return {"out": out}
    return {"out": out, **{"d" + x: d for x, d in zip(names, grads)}}


def _exact_muon(case, s):
    x = s["g"].double()
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + NS_EPS)
    for _ in range(5):
        if case["rows"] > case["cols"]:
            a = torch.bmm(x.mT.contiguous(), x)
            x = NS_A * x + torch.bmm(x, NS_B * a + NS_C * torch.bmm(a, a))
        else:
            a = torch.bmm(x, x.mT.contiguous())
            x = NS_A * x + torch.bmm(NS_B * a + NS_C * torch.bmm(a, a), x)
    return {"out": x}


def exact(case, seed):
    s = prepare(case, seed)
    form = {"embed": _exact_embed, "attn": _exact_attn, "muon": _exact_muon}
    return form[case["op"]](case, s)
