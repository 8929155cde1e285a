"""What is measured of the layer operators: attention over packed proteins (sliding window, first tokens that stay
visible, learned relative position bias, few queries over long keys) and the per-head norm of queries and keys with the
position rotation.  ``own`` false computes them in elementary torch operations in 32 bits, ``own`` true calls
``deepptmpred_amd.layers``.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def _norm(name, kind, dtype, rows, heads, kv_heads, dim, interleaved=False, restart=1024):
    return {"name": name, "op": "norm", "kind": kind, "dtype": dtype, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "interleaved": interleaved, "restart": restart}


def _attn(name, kind, dtype, seqs, longest, heads, kv_heads, dim, left=-1, right=-1, sinks=0, buckets=0, reach=0, few=0,
          ragged=True, empty=False):
    return {"name": name, "op": "attn", "kind": kind, "dtype": dtype, "seqs": seqs, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "left": left, "right": right, "sinks": sinks, "buckets": buckets,
            "reach": reach, "few": few, "ragged": ragged, "empty": empty}


def listed():
    return [
        # one protein of 480 residues and its two end tokens, 20 heads of 64 (rows of 1280): a call that waits for latency
        _norm("norm_one_protein", "forward", "bf16", 482, 20, 20, 64),
        # one new token of each of 64 sequences, shared key heads, neighbouring pairs
        _norm("norm_new_tokens", "forward", "f16", 64, 32, 8, 128, interleaved=True, restart=1),
        # a training batch of 64 pieces of 1024 tokens and a rest, forward and backward
        _norm("norm_batch_train", "train", "bf16", 65539, 20, 20, 64),
        # the same in the framework's default type, odd row count, shared key heads
        _norm("norm_f32_train", "train", "f32", 8191, 12, 4, 32, restart=441),
        # one protein of 480 residues and its two ends, with the relative bias: latency
        _attn("attn_one_protein", "forward", "bf16", 1, 482, 20, 20, 64, buckets=32, reach=128, ragged=False),
        # the site classifier's own windows: 51 rows, 4 heads of 16, fp32, trained with the bias in place of a position table
        _attn("attn_windows_train", "train", "f32", 2048, 51, 4, 4, 16, buckets=32, reach=50, ragged=False),
        # a ragged training batch of proteins, pieces of at most 1022 residues and two ends
        _attn("attn_proteins_train", "train", "bf16", 48, 1024, 20, 20, 64, buckets=32, reach=128, empty=True),
        # one long protein, 512 residues to either side and the first token: training
        _attn("attn_long_window_train", "train", "f16", 1, 16001, 8, 8, 64, left=512, right=512, sinks=1, buckets=32,
              reach=128, ragged=False),
        # long prompts that look back only, shared key heads of 128
        _attn("attn_causal_long", "forward", "bf16", 2, 8192, 16, 4, 128, right=0, ragged=False),
        # the 53 sites of one long protein: only their rows are needed, each over all residues
        _attn("attn_sites_long", "few", "f16", 1, 34003, 20, 20, 64, buckets=32, reach=128, few=53, ragged=False),
        # one new token of each of 64 sequences over caches up to 16,384 long, a window of 4,096 and four first tokens
        _attn("attn_new_tokens", "few", "bf16", 64, 16384, 32, 8, 128, left=4095, right=0, sinks=4, few=1, empty=True),
        # the sites of a few short proteins in the framework's default type
        _attn("attn_sites_f32", "few", "f32", 5, 441, 20, 20, 64, few=36),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([(20, 1), (4, 1), (12, 1), (4, 3), (8, 4), (4, 2)])
    heads = kv_heads * group
    if rng.random() < 0.35:
        most = 65539 * 1280 * 2 // (heads * dim * SIZES[dtype])
        return _norm(None, rng.choice(["forward", "train"]), dtype, spread(1, min(65539, most)), heads, kv_heads, dim,
                     rng.random() < 0.5, rng.choice([1, 51, 441, 1024]))
    left, right, sinks = rng.choice([(-1, -1, 0), (-1, -1, 0), (-1, 0, 0), (64, 64, 1), (512, 512, 1), (1023, 0, 4),
                                     (255, 0, 0), (0, 0, 0), (100, -1, 3)])
    buckets, reach = rng.choice([(0, 0), (0, 0), (32, 128), (16, 50), (64, 1000)])
    kind = rng.choice(["forward", "train", "few"])
    if kind == "train" and (left, right) == (0, 0):
        left = 31      # a row that sees one key alone has no gradient but rounding
    # the cost of a case in the plain form goes with seqs * heads * rows * longest
    most = 1.2e9 if kind == "train" else 1.6e9
    if kind == "few":
        seqs, few = rng.choice([(1, 1), (1, 53), (3, 36), (7, 1), (64, 1), (16, 5)])
        longest = spread(1, min(34003, int(5.0e7 / (seqs * kv_heads)), int(2.5e9 / (seqs * kv_heads * dim * 4))))
    else:
        longest, few = spread(32 if kind == "train" else 1, 8192), 0
        seqs = max(1, min(2048, int(most / (heads * longest * longest)), int(262144 / longest)))
        seqs = spread(1, seqs)
        while seqs * heads * longest * longest > most:
            longest = longest * 3 // 4
    return _attn(None, kind, dtype, seqs, max(1, longest), heads, kv_heads, dim, left, right, sinks, buckets, reach, few,
                 rng.random() < 0.7, rng.random() < 0.3)


def _lengths(case):
    """Rows and keys of every sequence; the same for every seed."""
    n, longest = case["seqs"], case["longest"]
    keys = np.full(n, longest, np.int64)
    if case["ragged"] and n > 1:
        r = np.random.RandomState(n * 31 + longest)
        keys = np.maximum(1, np.exp(r.uniform(math.log(max(1.0, longest / 12.0)), math.log(longest), n)).astype(np.int64))
        keys[n // 2] = longest
        keys[n - 1] = 1
    if case["empty"]:
        keys = np.insert(keys, n // 3, 0)
    rows = np.minimum(keys, case["few"]) if case["few"] > 1 else np.ones_like(keys) if case["few"] else keys.copy()
    return rows, keys


def _positions(case, rows, keys):
    """Where the queries stand: sites spread over the protein, otherwise the last rows."""
    out = [np.arange(a) + k - a if case["few"] < 2 else (np.arange(a) * k + k // 2) // max(1, a) for a, k in zip(rows, keys)]
    return np.concatenate(out).astype(np.int32) if out else np.zeros(0, np.int32)


def _visible(case, rows, keys):
    """Pairs of a query and a key that it sees, and the keys that some query sees."""
    pos, pairs, seen, at = _positions(case, rows, keys), 0, 0, 0
    for a, k in zip(rows, keys):
        p = pos[at:at + a].astype(np.int64)
        at += a
        if not a or not k:
            continue
        hi = np.full_like(p, k) if case["right"] < 0 else np.clip(p + case["right"] + 1, 0, k)
        lo = np.zeros_like(p) if case["left"] < 0 else np.maximum(p - case["left"], 0)
        lo = np.minimum(lo, hi)
        first = np.minimum(np.minimum(case["sinks"], hi), lo)
        pairs += int((hi - lo + first).sum())
        mark = np.zeros(k + 1, np.int64)
        np.add.at(mark, lo, 1)
        np.add.at(mark, hi, -1)
        mark = np.cumsum(mark)[:k] > 0
        mark[:int(first.max())] = True
        seen += int(mark.sum())
    return pairs, seen


def _bucket_map(n, reach, both):
    """Bucket of every distance j - p from -reach to reach: half of a side's buckets one distance each, the others by
    the logarithm of the distance, in whole numbers."""
    side = n // 2 if both else n
    near = side // 2
    steps = side - near
    ends = [d for d in range(near)]
    out = np.zeros(2 * reach + 1, np.int32)
    for d in range(reach + 1):
        b = d
        if d >= near:
            b = near
            while b + 1 < side and d ** steps >= near ** (steps - (b + 1 - near)) * reach ** (b + 1 - near):
                b += 1
        out[reach - d] = b
        out[reach + d] = b + (side if both and d else 0) if both else (b if not d else 0)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*size, by=1.0):
        return (torch.randn(*size, generator=g, device="cuda") * by).to(t)

    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "norm":
        n = case["rows"]
        x = normal(n, h + 2 * hk, d, by=1.5)
        s["q"], s["k"] = x[:, :h], x[:, h:h + hk]
        s["q_gain"] = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
        s["k_gain"] = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
        last = 20011
        s["positions"] = (torch.arange(n, device="cuda") % case["restart"]).to(torch.int32)
        if case["restart"] == 1:
            s["positions"] = torch.randint(0, last, (n,), generator=g, device="cuda", dtype=torch.int32)
        angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["kind"] == "train":
            s["dq2"], s["dk2"] = normal(n, h, d), normal(n, hk, d)
        return s
    rows, keys = _lengths(case)
    nq, nk = int(rows.sum()), int(keys.sum())
    if case["few"]:
        s["q"], s["k"], s["v"] = normal(nq, h, d), normal(nk, hk, d), normal(nk, hk, d)
    else:
        x = normal(nq, h + 2 * hk, d)
        s["q"], s["k"], s["v"] = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    s["table"] = s["buckets"] = None
    if case["buckets"]:
        s["table"] = normal(case["buckets"], h, by=0.7)
        s["buckets"] = torch.from_numpy(_bucket_map(case["buckets"], case["reach"], case["right"] != 0)).cuda()
    if case["kind"] == "train":
        s["dout"] = normal(nq, h, d)
    pos = _positions(case, rows, keys)
    # the layout that the padded form keeps: which packed row stands where, and back
    s["q_at"], s["q_back"] = _padding(rows)
    s["k_at"], s["k_back"] = _padding(keys)
    s["q_pos"] = torch.from_numpy(pos).cuda().long()
    s["k_len"] = torch.from_numpy(keys).cuda()
    if own:
        from deepptmpred_amd import layers
        s["plan"] = layers.AttentionPlan(rows, keys, heads=h, kv_heads=hk, head_dim=d, window=(case["left"], case["right"]),
                                         sinks=case["sinks"], q_positions=pos if case["few"] > 1 else None, training=case["kind"] == "train")
    return s


def _padding(lengths):
    """Packed row of every place of a [sequences, longest] block (the row behind the last where it holds none), and the
    place of every packed row."""
    longest = max(1, int(lengths.max()))
    start = np.cumsum(lengths) - lengths
    col = np.arange(longest)[None]
    at = np.where(col < lengths[:, None], start[:, None] + col, int(lengths.sum()))
    back = np.flatnonzero((col < lengths[:, None]).reshape(-1))
    return torch.from_numpy(at).cuda(), torch.from_numpy(back).cuda()


def _block(x, at, group):
    """[rows, heads, dim] -> [sequences * kv heads * group, longest, dim] in 32 bits; zeros where no row stands."""
    x = torch.cat([x.float(), torch.zeros_like(x[:1], dtype=torch.float32) if x.shape[0] else
                   torch.zeros((1,) + x.shape[1:], device=x.device)])[at]
    return x.permute(0, 2, 1, 3).repeat_interleave(group, 1).flatten(0, 1).contiguous()


def _packed(x, back, heads):
    """The way back from _block."""
    return x.unflatten(0, (-1, heads)).permute(0, 2, 1, 3).flatten(0, 1)[back]


def _scores(s):
    """Scaled and biased scores [sequences * heads, rows, keys], -inf where the key is not visible."""
    c = s["case"]
    g = c["heads"] // c["kv_heads"]
    q, k = _block(s["q"], s["q_at"], 1), _block(s["k"], s["k_at"], g)
    x = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(c["dim"] ** -0.5).unflatten(0, (-1, c["heads"]))
    pos = torch.cat([s["q_pos"], s["q_pos"].new_zeros(1)])[s["q_at"]]
    far = torch.arange(k.shape[1], device=q.device) - pos[..., None]
    key = torch.arange(k.shape[1], device=q.device)
    see = (key < s["k_len"][:, None])[:, None] & (s["q_at"] < s["q"].shape[0])[..., None]
    if c["right"] >= 0:
        see = see & (far <= c["right"])
    if c["left"] >= 0:
        see = see & ((far >= -c["left"]) | (key < c["sinks"]))
    if c["buckets"]:
        r = c["reach"]
        of = s["buckets"].long()[far.clamp(-r, r) + r]
        x = x + s["table"].float()[of].permute(0, 3, 1, 2)
    return x.masked_fill_(~see[:, None], -math.inf), q, k


def _softmax(x):
    m = x.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    p = (x - m).exp_()
    z = p.sum(-1, keepdim=True)
    return p.div_(torch.where(z > 0, z, torch.ones_like(z))), (z.log() + m)[..., 0]


def _plain_attention(s):
    c = s["case"]
    h, hk = c["heads"], c["kv_heads"]
    g = h // hk
    x, q, k = _scores(s)
    p, lse = _softmax(x)
    del x
    v = _block(s["v"], s["k_at"], g)
    p = p.flatten(0, 1)
    t = s["q"].dtype
    o = torch.bmm(p, v)
    found = {"out": _packed(o, s["q_back"], h).to(t),
             "lse": lse.permute(1, 0, 2).flatten(1)[:, s["q_back"]]}
    if c["kind"] != "train":
        return found
    do = _block(s["dout"], s["q_at"], 1)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
    ds = torch.bmm(do, v.transpose(1, 2).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    scale = c["dim"] ** -0.5
    found["dq"] = (_packed(torch.bmm(ds, k), s["q_back"], h) * scale).to(t)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q) * scale
    found["dk"] = _packed(dk.unflatten(0, (-1, g)).sum(1), s["k_back"], hk).to(t)
    found["dv"] = _packed(dv.unflatten(0, (-1, g)).sum(1), s["k_back"], hk).to(t)
    if c["buckets"]:
        # sums along the diagonals (the same distance), then of the distances of a bucket
        n, r = ds.shape[-1], c["reach"]
        ds = ds.unflatten(0, (-1, h)).sum(0).flip(1)
        ds = torch.cat([ds, torch.zeros_like(ds)], 2).flatten(1)[:, :-n].unflatten(1, (n, 2 * n - 1)).double().sum(1)
        of = s["buckets"].long()[torch.arange(1 - n, n, device=ds.device).clamp(-r, r) + r]
        one = (of[:, None] == torch.arange(c["buckets"], device=ds.device)).double()
        found["dtable"] = (ds @ one).T.to(t)
    return found


def _pairs(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _joined(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _plain_norm_one(s, x, gain, dy):
    c = s["case"]
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    t, x = x.dtype, x.float()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    a, b = _pairs(x * r * gain, c["interleaved"])
    y = _joined(a * cos - b * sin, b * cos + a * sin, c["interleaved"]).to(t)
    if dy is None:
        return y, None, None
    a, b = _pairs(dy.float(), c["interleaved"])
    d = _joined(a * cos + b * sin, b * cos - a * sin, c["interleaved"])
    dgain = (d * x * r).double().sum((0, 1)).float()
    d = d * gain
    return y, (r * (d - x * r * r * (d * x).mean(-1, keepdim=True))).to(t), dgain


def run(state):
    s, c = state, state["case"]
    if own:
        from deepptmpred_amd import layers
        if c["op"] == "norm":
            more = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], positions=s["positions"], eps=EPS, interleaved=c["interleaved"])
            q, k = layers.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], **more)
            found = {"q": q, "k": k}
            if c["kind"] == "train":
                found["dq"], found["dk"], found["dq_gain"], found["dk_gain"] = layers.qk_norm_rope_backward(
                    s["dq2"], s["dk2"], s["q"], s["k"], s["cos"], s["sin"], **more)
            return found
        out, lse = layers.attention(s["q"], s["k"], s["v"], s["plan"], table=s["table"], buckets=s["buckets"])
        found = {"out": out, "lse": lse}
        if c["kind"] == "train":
            found["dq"], found["dk"], found["dv"], dtable = layers.attention_backward(
                s["dout"], s["q"], s["k"], s["v"], out, lse, s["plan"], table=s["table"], buckets=s["buckets"])
            if c["buckets"]:
                found["dtable"] = dtable
        return found
    if c["op"] == "attn":
        return _plain_attention(s)
    train = c["kind"] == "train"
    q, dq, dgq = _plain_norm_one(s, s["q"], s["q_gain"], s["dq2"] if train else None)
    k, dk, dgk = _plain_norm_one(s, s["k"], s["k_gain"], s["dk2"] if train else None)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dq_gain": dgq, "dk_gain": dgk} if train else {"q": q, "k": k}


def work(case):
    h, hk, d, size = case["heads"], case["kv_heads"], case["dim"], SIZES[case["dtype"]]
    train = case["kind"] == "train"
    if case["op"] == "norm":
        n = case["rows"]
        data = n * (h + hk) * d
        # the angles of the positions that occur, and the positions
        angles = min(n, max(case["restart"], 1 if case["restart"] > 1 else n)) * d * 4 + n * 4
        return {"bytes": data * size * (5 if train else 2) + angles + 2 * d * 4 * (2 if train else 1),
                "flops": data * (30 if train else 10)}
    rows, keys = _lengths(case)
    pairs, seen = _visible(case, rows, keys)
    nq, nk = int(rows.sum()), int(keys.sum())
    bytes_ = 2 * nq * h * d * size + 2 * seen * hk * d * size + nq * h * 4 + case["buckets"] * h * size
    flops = 4 * d * pairs * h
    if train:
        # the gradient of the output in, three gradients out
        bytes_ += 2 * nq * h * d * size + 2 * nk * hk * d * size + case["buckets"] * h * size
        flops += 10 * d * pairs * h
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    train = case["kind"] == "train"
    if case["op"] == "norm":
        found = {}
        f = 10000.0 ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
        # (rows, 1, dim / 2) unit numbers e^(i angle)
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                           s["positions"].double()[:, None, None] * f)
        for name in ("q", "k"):
            x, gain = s[name].double(), s[name + "_gain"].double()
            z = (x * gain) / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()

            def turned(y, by):
                if case["interleaved"]:
                    y = torch.view_as_complex(y.unflatten(-1, (d // 2, 2)).contiguous()) * by
                    return torch.view_as_real(y).flatten(-2)
                y = torch.complex(y[..., :d // 2], y[..., d // 2:]) * by
                return torch.cat([y.real, y.imag], -1)

            found[name] = turned(z, turn)
            if train:
                dz = turned(s["d" + name + "2"].double(), turn.conj())
                ms = x.pow(2).mean(-1, keepdim=True) + EPS
                found["d" + name] = dz * gain / ms.sqrt() - x * (dz * gain * x).sum(-1, keepdim=True) / (d * ms.pow(1.5))
                found["d" + name + "_gain"] = (dz * x / ms.sqrt()).flatten(0, 1).sum(0)
        order = ["q", "k", "dq", "dk", "dq_gain", "dk_gain"] if train else ["q", "k"]
        return {n: found[n] for n in order}
    rows, keys = _lengths(case)
    if int((rows * keys).sum()) * h > 4e9:
        return None
    out = torch.zeros(int(rows.sum()), h, d, device="cuda", dtype=torch.float64)
    lse = torch.full((h, int(rows.sum())), -math.inf, device="cuda", dtype=torch.float64)
    dq = torch.zeros_like(out)
    dk = torch.zeros(int(keys.sum()), hk, d, device="cuda", dtype=torch.float64)
    dv = torch.zeros_like(dk)
    dtable = torch.zeros(max(1, case["buckets"]), h, device="cuda", dtype=torch.float64)
    pos = s["q_pos"]
    # sequences of one shape at the same positions go together
    shapes, a0, k0 = {}, 0, 0
    for a, k in zip(rows.tolist(), keys.tolist()):
        if a and k:
            shapes.setdefault((a, k), []).append((a0, k0))
        a0, k0 = a0 + a, k0 + k
    for (a, k), where in shapes.items():
        qi = torch.tensor([[w[0] + i for i in range(a)] for w in where], device="cuda") if len(where) > 1 else \
            torch.arange(where[0][0], where[0][0] + a, device="cuda")[None]
        ki = torch.tensor([[w[1] + i for i in range(k)] for w in where], device="cuda") if len(where) > 1 else \
            torch.arange(where[0][1], where[0][1] + k, device="cuda")[None]
        p = pos[qi[0]]
        j = torch.arange(k, device="cuda")
        hidden = torch.zeros(a, k, dtype=torch.bool, device="cuda")
        if case["right"] >= 0:
            hidden |= j[None] > p[:, None] + case["right"]
        if case["left"] >= 0:
            hidden |= (j[None] < p[:, None] - case["left"]) & (j[None] >= case["sinks"])
        if case["buckets"]:
            r = case["reach"]
            bucket = s["buckets"].long()[(j[None] - p[:, None]).clamp(-r, r) + r]
        for n in range(h):
            m = n // (h // hk)
            qh, kh, vh = s["q"][qi, n].double(), s["k"][ki, m].double(), s["v"][ki, m].double()
            z = torch.matmul(qh, kh.mT.contiguous()) / math.sqrt(d)
            if case["buckets"]:
                z += s["table"][:, n].double()[bucket]
            z.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(z, -1)
            w = torch.exp(z - torch.where(total > -math.inf, total, torch.zeros_like(total))[..., None])
            y = torch.matmul(w, vh)
            out[qi, n] = y
            lse[n][qi] = total
            if train:
                dy = s["dout"][qi, n].double()
                dw = torch.matmul(dy, vh.mT.contiguous())
                dz = w * (dw - (w * dw).sum(-1, keepdim=True))
                dq[qi, n] = torch.matmul(dz, kh) / math.sqrt(d)
                dk[ki, m] += torch.matmul(dz.mT.contiguous(), qh) / math.sqrt(d)
                dv[ki, m] += torch.matmul(w.mT.contiguous(), dy)
                if case["buckets"]:
                    both = dz.sum(0)
                    # by distance first: a row's own order, shifted by its position
                    width = a + k - 1
                    by = torch.zeros(width, a, device="cuda", dtype=torch.float64)
                    i = torch.arange(a, device="cuda")
                    by[(j[None] - i[:, None] + a - 1), i[:, None].expand(a, k)] = both
                    of = torch.full((width,), 0, device="cuda", dtype=torch.long)
                    of[(j[None] - i[:, None] + a - 1).flatten()] = bucket.flatten()
                    dtable[:, n].index_add_(0, of, by.sum(1))
    found = {"out": out, "lse": lse}
    if train:
        found |= {"dq": dq, "dk": dk, "dv": dv}
        if case["buckets"]:
            found["dtable"] = dtable
    return found
