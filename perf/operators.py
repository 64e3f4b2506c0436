"""Training operators on ragged batches, as cases to be measured: one forward and backward pass of

    layer_norm   over the rows of packed sequences, with the gradients of the input, the weight and the bias
    embedding    of sequences of token indices, scaled, with the dense gradient of the table
    attention    of every sequence over itself (one packed q|k|v matrix) or over the sequence of the same number of another
                 batch (separate q, k, v), with the gradients of q, k and v; the probabilities are computed again

A batch is B sequences of L_i rows, concatenated without padding: T = sum(L_i).  The lengths belong to the case (they are
drawn from its own number "lengths"), the values to the seed.

Where `own` is true `run` calls nestedtensor_b200, otherwise it computes the same results from elementary torch operations in
32 bits: the attention pads the batch to (B, L_max), as a program without ragged kernels does.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # -- layer norm ---------------------------------------------------------------------------------------------
        # 64 short sequences of 256 features in 32 bits: the smallest batch of the benchmark configurations, latency counts
        dict(name="norm_small_fp32", op="norm", dtype="fp32", batch=64, dist="uniform", lo=1, hi=128, features=256, lengths=1),
        # a width that no 16-byte vector divides, as after a concatenation of features
        dict(name="norm_odd_bf16", op="norm", dtype="bf16", batch=96, dist="uniform", lo=1, hi=511, features=771, lengths=2),
        # the batch of the base-size encoder: 128 sequences of 32 to 512 tokens, 768 features
        dict(name="norm_base_fp16", op="norm", dtype="fp16", batch=128, dist="uniform", lo=32, hi=512, features=768, lengths=3),
        # the largest batch of the benchmark configurations: 4096 log-normal lengths, 1024 features, about a million tokens
        dict(name="norm_large_bf16", op="norm", dtype="bf16", batch=4096, dist="lognormal", lo=1, hi=1024, features=1024, lengths=4),
        # -- embedding ----------------------------------------------------------------------------------------------
        # a few sentences against a small table: latency
        dict(name="embed_small_fp32", op="embed", dtype="fp32", batch=8, dist="uniform", lo=1, hi=64, features=256, vocab=1000, padding=False, lengths=5),
        # odd table width, a padding index among the tokens
        dict(name="embed_odd_fp16", op="embed", dtype="fp16", batch=100, dist="uniform", lo=1, hi=300, features=333, vocab=8191, padding=True, lengths=6),
        # the large encoder's batch: 1024 sequences, 70 % short and 30 % long, table of 50 000 tokens
        dict(name="embed_large_bf16", op="embed", dtype="bf16", batch=1024, dist="mixed", lo=16, hi=512, features=1024, vocab=50000, padding=True, lengths=7),
        # -- attention ----------------------------------------------------------------------------------------------
        # four very short sequences: latency
        dict(name="attend_small_bf16", op="attend", dtype="bf16", batch=4, dist="uniform", lo=1, hi=40, heads=16, head_dim=64, cross=False, lengths=8),
        # queries over the sequences of another batch in 32 bits, some of them empty
        dict(name="attend_cross_fp32", op="attend", dtype="fp32", batch=16, dist="uniform", lo=0, hi=200, heads=4, head_dim=64, cross=True, lengths=9),
        # the base-size encoder's batch: 12 heads of 64, 32 to 512 tokens
        dict(name="attend_base_fp16", op="attend", dtype="fp16", batch=128, dist="uniform", lo=32, hi=512, heads=12, head_dim=64, cross=False, lengths=10),
        # a quarter of the large encoder's batch: 16 heads of 64, 70 % short and 30 % long sequences
        dict(name="attend_large_bf16", op="attend", dtype="bf16", batch=256, dist="mixed", lo=16, hi=512, heads=16, head_dim=64, cross=False, lengths=11),
        # two long documents of odd lengths, heads of 128: few rows of work items, a long axis
        dict(name="attend_long_bf16", op="attend", dtype="bf16", batch=2, dist="uniform", lo=2500, hi=5000, heads=8, head_dim=128, cross=False, lengths=12),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "embed", "attend"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    case = dict(op=op, dtype=dtype, lengths=rng.randrange(1 << 30))
    if op == "attend":
        case["head_dim"] = rng.choice([32, 64, 64, 64, 128])
        case["heads"] = rng.randint(1, 16)
        hi = _spread(rng, 8, 4000)
        # the padded work of the plain form, heads * head_dim * batch * hi^2, stays under that of the largest listed case
        most = max(1, int(6.5e10 / (8 if dtype == "fp32" else 1) / (case["heads"] * case["head_dim"] * hi * hi)))
        case.update(batch=_spread(rng, 1, min(most, 512)), dist=rng.choice(["uniform", "mixed"]), lo=rng.choice([0, 1, 1 + hi // 4]),
                    hi=hi, cross=rng.random() < 0.4)
    else:
        features = _spread(rng, 32, 4096)
        if rng.random() < 0.6:
            features = max(32, features // 32 * 32)
        hi = _spread(rng, 8, 2000)
        most = max(1, int((9.0e8 if op == "norm" else 1.5e8) / (features * hi)))
        case.update(batch=_spread(rng, 1, min(most, 8192)), dist=rng.choice(["uniform", "lognormal", "mixed"]), lo=rng.choice([0, 1, 1 + hi // 8]),
                    hi=hi, features=features)
        if op == "embed":
            case.update(vocab=_spread(rng, 100, min(65536, 60_000_000 // features)), padding=rng.random() < 0.5)
    return case


def _lengths(case, key_side=False):
    """The B lengths of the case: uniform in [lo, hi]; log-normal about 200 (or hi / 4), clipped; or 70 % up to a quarter of hi
    and 30 % above.  The keys of a cross attention have lengths of their own."""
    rng = random.Random(case["lengths"] * 2 + key_side)
    lo, hi = case["lo"], case["hi"]
    out = []
    for _ in range(case["batch"]):
        if case["dist"] == "uniform":
            n = rng.randint(lo, hi)
        elif case["dist"] == "lognormal":
            n = int(round(math.exp(math.log(max(1.0, min(200.0, hi / 4))) + 0.6 * rng.gauss(0, 1))))
        else:
            n = rng.randint(lo, max(lo, hi // 4)) if rng.random() < 0.7 else rng.randint(max(lo, hi // 4), hi)
        out.append(max(lo, min(hi, n)))
    if sum(out) == 0:
        out[0] = 1
    return out


# ------------------------------------------------------------------ what a program has in hand
def _ragged(lengths, features):
    """(sizes on the host, [element offsets | sizes] on the GPU) of sequences (L_i, features), or (L_i,) where features is None."""
    n = torch.tensor(lengths, dtype=torch.int64)
    cols = [n] if features is None else [n, torch.full_like(n, features)]
    sizes = torch.stack(cols, 1).contiguous()
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(sizes.prod(1), 0)])
    return sizes, torch.cat([offsets, sizes.reshape(-1)]).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + case["lengths"])
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    lengths = _lengths(case)
    T = sum(lengths)
    state = dict(case=case)
    if case["op"] == "norm":
        F = case["features"]
        state["sizes"], state["meta"] = _ragged(lengths, F)
        # activations with a mean and a spread of their own in every row, as after a residual stream of several layers
        x = normal(T, F)
        x.mul_(torch.exp(0.5 * torch.randn(T, 1, generator=g, device="cuda")).to(dtype)).add_(normal(T, 1, std=0.5))
        state.update(x=x.requires_grad_(), weight=normal(F, std=0.1, mean=1.0).requires_grad_(), bias=normal(F, std=0.1).requires_grad_(),
                     grad=normal(T, F, std=0.1), eps=1e-5)
    elif case["op"] == "embed":
        F, V = case["features"], case["vocab"]
        state["sizes"], state["meta"] = _ragged(lengths, None)
        # token frequencies fall off as in text: the k-th most frequent about as 1 / k; which tokens those are is shuffled
        u = torch.rand(T, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.clamp(torch.exp(u * math.log(V + 1.0)).long() - 1, 0, V - 1)
        index = torch.randperm(V, generator=g, device="cuda")[rank]
        state.update(index=index, weight=normal(V, F, std=0.05).requires_grad_(), grad=normal(T, F, std=0.1), scale=math.sqrt(F),
                     padding=int(index[0]) if case["padding"] else None)
    else:
        E = case["heads"] * case["head_dim"]
        state["scaling"] = case["head_dim"] ** -0.5
        state["grad"] = normal(T, E, std=0.1)
        state["longest"] = max(lengths)
        if case["cross"]:
            keys = _lengths(case, True)
            state["sizes"], state["meta"] = _ragged(lengths, E)
            state["key_sizes"], state["key_meta"] = _ragged(keys, E)
            state["key_longest"] = max(keys)
            state.update(q=normal(T, E).requires_grad_(), k=normal(sum(keys), E).requires_grad_(), v=normal(sum(keys), E).requires_grad_())
        else:
            state["sizes"], state["meta"] = _ragged(lengths, 3 * E)
            state["qkv"] = normal(T, 3 * E).requires_grad_()
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "embed": _own_embed, "attend": _own_attend}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "embed": _plain_embed, "attend": _plain_attend}[op](state)


def _own_norm(s):
    import nestedtensor_b200 as nestedtensor
    x, w, b = s["x"], s["weight"], s["bias"]
    nt = nestedtensor.NestedTensor(x.view(-1), s["sizes"], s["meta"])
    y = nestedtensor.nn.training.layer_norm(nt, (x.size(1),), w, b, s["eps"]).values()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["grad"])
    return {"out": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_embed(s):
    import nestedtensor_b200 as nestedtensor
    nt = nestedtensor.NestedTensor(s["index"], s["sizes"], s["meta"])
    y = nestedtensor.nn.training.embedding(nt, s["weight"], padding_idx=s["padding"], scale=s["scale"]).values()
    dw, = torch.autograd.grad(y, (s["weight"],), s["grad"])
    return {"out": y.detach(), "dweight": dw}


def _own_attend(s):
    import nestedtensor_b200 as nestedtensor
    heads, training = s["case"]["heads"], nestedtensor.nn.training
    if not s["case"]["cross"]:
        nt = nestedtensor.NestedTensor(s["qkv"].view(-1), s["sizes"], s["meta"])
        y = training.self_attention(nt, heads, s["scaling"]).values()
        dqkv, = torch.autograd.grad(y, (s["qkv"],), s["grad"])
        return {"out": y.detach(), "dqkv": dqkv}
    q = nestedtensor.NestedTensor(s["q"].view(-1), s["sizes"], s["meta"])
    k = nestedtensor.NestedTensor(s["k"].view(-1), s["key_sizes"], s["key_meta"])
    v = nestedtensor.NestedTensor(s["v"].view(-1), s["key_sizes"], s["key_meta"])
    y = training.attention(q, k, v, heads, s["scaling"]).values()
    dq, dk, dv = torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["grad"])
    return {"out": y.detach(), "dq": dq, "dk": dk, "dv": dv}


def _plain_norm(s):
    x, w, g = s["x"].float(), s["weight"].float(), s["grad"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + s["eps"])
    n = d * rstd
    gw = g * w
    dx = (gw - gw.mean(1, keepdim=True) - n * (gw * n).mean(1, keepdim=True)) * rstd
    t = s["x"].dtype
    return {"out": (n * w + s["bias"].float()).to(t), "dx": dx.to(t), "dweight": (g * n).sum(0).to(t), "dbias": g.sum(0).to(t)}


def _plain_embed(s):
    w, index = s["weight"], s["index"]
    out = (w[index].float() * s["scale"]).to(w.dtype)
    dw = torch.zeros(w.shape, device=w.device)
    dw.index_add_(0, index, s["grad"].float() * s["scale"])
    if s["padding"] is not None:
        dw[s["padding"]] = 0
    return {"out": out, "dweight": dw.to(w.dtype)}


class _Padding:
    """Packed rows to (B, L, ...) and back, by indices made on the GPU."""

    def __init__(self, meta, batch, row_elems, tokens, longest):
        starts = torch.div(meta[:batch + 1], row_elems, rounding_mode="floor")
        pos = torch.arange(longest, device=meta.device)
        self.valid = pos[None, :] < (starts[1:] - starts[:-1])[:, None]
        self.rows = torch.clamp(starts[:-1, None] + pos[None, :], max=max(tokens - 1, 0))
        t = torch.arange(tokens, device=meta.device)
        b = torch.searchsorted(starts, t, right=True) - 1
        self.back = b * longest + (t - starts[b])

    def pad(self, x, heads):  # [T, H*d] -> [B, H, L, d]
        if x.size(0) == 0:
            x = x.new_zeros(1, x.size(1))
        y = torch.where(self.valid[:, :, None], x[self.rows].float(), 0.0)
        return y.view(y.size(0), y.size(1), heads, -1).transpose(1, 2)

    def unpad(self, y):
        y = y.transpose(1, 2)
        return y.reshape(y.size(0) * y.size(1), -1)[self.back]


def _plain_attend(s):
    case = s["case"]
    H, E, B = case["heads"], case["heads"] * case["head_dim"], case["batch"]
    if case["cross"]:
        q, k, v = s["q"], s["k"], s["v"]
        pq = _Padding(s["meta"], B, E, q.size(0), s["longest"])
        pk = _Padding(s["key_meta"], B, E, k.size(0), s["key_longest"])
    else:
        q, k, v = s["qkv"].split(E, 1)
        pq = pk = _Padding(s["meta"], B, 3 * E, q.size(0), s["longest"])
    qp, kp, vp, gp = pq.pad(q, H), pk.pad(k, H), pk.pad(v, H), pq.pad(s["grad"], H)
    p = torch.matmul(qp, kp.transpose(2, 3)).mul_(s["scaling"])
    p.masked_fill_(~pk.valid[:, None, None, :], -math.inf)
    top = p.amax(3, keepdim=True) if p.size(3) else p.new_zeros(p.shape[:3] + (1,))
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(3, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p, vp)
    dv = torch.matmul(p.transpose(2, 3), gp)
    ds = torch.matmul(gp, vp.transpose(2, 3)).sub_((gp * out).sum(3, keepdim=True)).mul_(p).mul_(s["scaling"])
    del p
    dq, dk = torch.matmul(ds, kp), torch.matmul(ds.transpose(2, 3), qp)
    t = q.dtype
    out, dq, dk, dv = pq.unpad(out).to(t), pq.unpad(dq).to(t), pk.unpad(dk).to(t), pk.unpad(dv).to(t)
    if case["cross"]:
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return {"out": out, "dqkv": torch.cat([dq, dk, dv], 1)}


# ------------------------------------------------------------------ the same in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        if case["op"] == "embed":
            return _exact_embed(s)
        return _exact_attend(s)


def _exact_norm(s):
    x = s["x"]
    T, F = x.shape
    w, b = s["weight"].double(), s["bias"].double()
    out, dx = torch.empty(T, F, dtype=torch.float64, device=x.device), torch.empty(T, F, dtype=torch.float64, device=x.device)
    dw, db = torch.zeros(F, dtype=torch.float64, device=x.device), torch.zeros(F, dtype=torch.float64, device=x.device)
    for r in range(0, T, 1 << 16):
        xr, g = x[r:r + (1 << 16)].double(), s["grad"][r:r + (1 << 16)].double()
        var, mean = torch.var_mean(xr, 1, unbiased=False, keepdim=True)
        std = torch.sqrt(var + s["eps"])
        n = (xr - mean) / std
        out[r:r + (1 << 16)] = n * w + b
        # the Jacobian of (x - mean) / std applied to g w: (I - 11'/F - nn'/F) / std
        gw = g * w
        dx[r:r + (1 << 16)] = (gw - gw.sum(1, keepdim=True) / F - n * ((n * gw).sum(1, keepdim=True) / F)) / std
        dw += torch.einsum("tf,tf->f", n, g)
        db += g.sum(0)
    return {"out": out, "dx": dx, "dweight": dw, "dbias": db}


def _exact_embed(s):
    w, index = s["weight"], s["index"]
    out = w.double()[index] * s["scale"]
    order = torch.argsort(index, stable=True)
    tokens, counts = torch.unique_consecutive(index[order], return_counts=True)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    # sums of the sorted rows as differences of running sums (which cost a few of the 16 digits), some columns at a time
    last = torch.cumsum(counts, 0)
    for c in range(0, w.size(1), 128):
        run_sum = torch.cumsum(s["grad"][:, c:c + 128].double()[order], 0)[last - 1]
        run_sum[1:] = run_sum[1:] - run_sum[:-1].clone()
        dw[tokens, c:c + 128] = run_sum * s["scale"]
    if s["padding"] is not None:
        dw[s["padding"]] = 0
    return {"out": out, "dweight": dw}


def _exact_attend(s):
    case = s["case"]
    H, d = case["heads"], case["head_dim"]
    E = H * d
    q, k, v = (s["q"], s["k"], s["v"]) if case["cross"] else s["qkv"].split(E, 1)
    lq = _lengths(case)
    lk = _lengths(case, True) if case["cross"] else lq
    out, dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in (q, q, k, v))
    a = c = 0
    for n, m in zip(lq, lk):
        rows, cols = slice(a, a + n), slice(c, c + m)
        a, c = a + n, c + m
        if n == 0 or m == 0:
            continue
        for h0 in range(0, H, 4):  # a few heads at a time: long sequences in 64 bits
            part = slice(h0 * d, min(H, h0 + 4) * d)
            Q, K, V, G = (x[r, part].double().view(-1, (part.stop - part.start) // d, d).transpose(0, 1)
                          for x, r in ((q, rows), (k, cols), (v, cols), (s["grad"], rows)))
            P = torch.softmax(torch.einsum("hid,hjd->hij", Q, K) * s["scaling"], 2)
            dP = torch.einsum("hid,hjd->hij", G, V)
            # the softmax's Jacobian with the sum over the probabilities themselves
            dS = P * (dP - (P * dP).sum(2, keepdim=True)) * s["scaling"]
            for to, r, y in ((out, rows, torch.einsum("hij,hjd->ihd", P, V)), (dq, rows, torch.einsum("hij,hjd->ihd", dS, K)),
                             (dk, cols, torch.einsum("hij,hid->jhd", dS, Q)), (dv, cols, torch.einsum("hij,hid->jhd", P, G))):
                to[r, part] = y.reshape(y.size(0), -1)
    if case["cross"]:
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return {"out": out, "dqkv": torch.cat([dq, dk, dv], 1)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    lengths = _lengths(case)
    T = sum(lengths)
    if case["op"] == "norm":
        F = case["features"]
        # the input read and the output written; then input and gradient read, the input's gradient written
        return {"bytes": 5 * T * F * size + 4 * F * size, "flops": 20 * T * F}
    if case["op"] == "embed":
        F, V = case["features"], case["vocab"]
        # rows gathered (a row used again is read once, so at most the table), written, their gradients read, the table's written
        return {"bytes": (min(T, V) + 2 * T + V) * F * size + 2 * T * 8, "flops": 2 * T * F}
    E = case["heads"] * case["head_dim"]
    keys = _lengths(case, True) if case["cross"] else lengths
    S = sum(keys)
    # q, k, v read and the output written; then q, k, v, the output and its gradient read, three gradients written; two products
    # of L_q x L_k x d a head forward, five backward
    return {"bytes": ((2 * T + 2 * S) + (3 * T + 2 * S) + (T + 2 * S)) * E * size,
            "flops": 14 * E * sum(n * m for n, m in zip(lengths, keys))}
