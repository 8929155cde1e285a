"""Layer operators on the GPU where values are what goes wrong: non-finite operands of pairs that do not count, rows of NaN, gradients
far from one.  Expected values are the float64 restatement's (oracle/layers_ref.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from deepptmpred_amd import layers  # noqa: E402
from oracle import layers_ref as R  # noqa: E402
from test_gpu_layers import attend, host, tensor, within  # noqa: E402

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def rows_within(t, want, name, keep):
    value, bound = want[name]
    within(t[torch.from_numpy(keep).cuda()], (value[keep], bound[keep]), name)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [64, 51, 32])
def test_short_sequences_with_a_hidden_value_row_that_is_not_finite(dtype, rows):
    """delta of the rows that see such a value is not finite; it reaches the keys those rows see, and the buckets of the distances
    in the window, and nothing else."""
    rng = np.random.default_rng(90)
    bad = (10, 11)
    q, k, v, dout = (tensor(rng, dtype, 2 * rows, 2, 32) for _ in range(4))
    window, lens = (5, 4), [rows, rows]
    b, table = layers.relative_buckets(8, 20), tensor(rng, dtype, 8, 2)
    plan = layers.AttentionPlan(lens, heads=2, head_dim=32, window=window)
    out, _ = layers.attention(q, k, v, plan, table=table, buckets=b)
    want = R.attention(host(q), host(k), host(v), lens, lens, window, 0, None, None, host(table), b.cpu().numpy(), host(dout), host(out), dtype)
    v2 = v.clone()
    v2[bad[0]], v2[bad[1], :, 3] = NAN, INF
    out2, lse2 = layers.attention(q, k, v2, plan, table=table, buckets=b)
    dq, dk, dv, dtable = layers.attention_backward(dout, q, k, v2, out2, lse2, plan, table=table, buckets=b)
    p, j = np.arange(2 * rows)[:, None], np.arange(2 * rows)[None]
    see = (j <= p + window[1]) & (j >= p - window[0]) & (p // rows == j // rows)
    met = see[:, list(bad)].any(1)
    rows_within(dq, want, "dq", ~met)
    touched = see[met].any(0)
    rows_within(dk, want, "dk", ~touched)
    assert not np.isfinite(host(dk)[touched]).all(axis=(1, 2)).any()
    within(dv, want["dv"], "dv")                    # the weights do not depend on values
    # distances -5 .. 4 take buckets 0, 1, 2 and 5, 6
    d = host(dtable)
    assert (d[[3, 7]] == 0).all() and np.isnan(d[[0, 1, 2, 5, 6]]).all()


# sequences, heads, dim, listed positions: the short backward kernel, the split forward kernel, the two wide ones
HIDING = [([51, 20], 2, 32, False), ([64], 2, 64, False), ([90, 33], 2, 32, False), ([90], 3, 64, True), ([70], 2, 128, False),
          ([200], 64, 32, False), ([256] * 4, 64, 16, False), ([256] * 4, 64, 64, True)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,heads,dim,given", HIDING)
def test_pairs_hidden_by_the_table_and_operands_that_are_not_finite(dtype, lens, heads, dim, given):
    """A table entry that hides its bucket hides it from NaN and infinities too, in both directions."""
    rng = np.random.default_rng(91)
    n = sum(lens)
    q, k, v, dout = (tensor(rng, dtype, n, heads, dim) for _ in range(4))
    b = layers.relative_buckets(8, 9)
    table = tensor(rng, dtype, 8, heads)
    table[[3, 7]] = -INF                             # distances of 5 and more (bucket 2: 2 to 4)
    table[:, heads - 1] = -INF                       # the last head sees nothing
    hidden = [3, 7]
    pos = R.default_positions(lens, lens).astype(np.int32)
    plan = layers.AttentionPlan(lens, heads=heads, head_dim=dim, q_positions=pos if given else None)

    def run(q, k, v, dout):
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        return (out, lse) + layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)

    plain = run(q, k, v, dout)
    names = ("out", "lse", "dq", "dk", "dv", "dtable")
    want = R.attention(host(q), host(k), host(v), lens, lens, (-1, -1), 0, None, None, host(table), b.cpu().numpy(), host(dout), host(plain[0]), dtype)
    for t, name in zip(plain, names):
        within(t, want[name], name)
    of = b.cpu().numpy()
    start = np.repeat(np.cumsum([0] + lens[:-1]), lens)
    see = (start[:, None] == start[None]) & ~np.isin(of[np.clip(np.arange(n)[None] - np.arange(n)[:, None], -9, 9) + 9], hidden)

    def rest(got, met_rows, met_keys, dv_keys):
        for t, name, keep in zip(got, names, (~met_rows, None, ~met_rows, ~met_keys, ~dv_keys)):
            if name == "lse":
                value, bound = want[name]
                within(t[:, torch.from_numpy(~met_rows).cuda()], (value[:, ~met_rows], bound[:, ~met_rows]), name)
            else:
                rows_within(t, want, name, keep)
        d = host(got[5])
        assert (d[hidden] == 0).all() and (d[:, heads - 1] == 0).all() and np.isnan(d[:, 0][[0, 1, 2, 5, 6]]).all()
        # the last head is empty whatever its operands hold
        assert not got[0][:, -1].any() and torch.isneginf(got[1][-1]).all() and not any(t[:, -1].any() for t in got[2:5])

    # keys of NaN and infinity, values of infinity
    k2, v2 = k.clone(), v.clone()
    k2[12], k2[13, :, 1], v2[13], v2[14] = NAN, INF, INF, -INF
    met = see[:, [12, 13, 14]].any(1)
    rest(run(q, k2, v2, dout), met, see[met].any(0), see[met].any(0))
    # a row of NaN, and a gradient of infinity
    q2, dout2 = q.clone(), dout.clone()
    q2[15], dout2[16] = NAN, INF
    met = np.isin(np.arange(n), (15, 16))
    got = run(q2, k, v, dout2)
    rest((plain[0], plain[1]) + got[2:], met, see[met].any(0), see[met].any(0))
    rows_within(got[0], want, "out", np.arange(n) != 15)
    rows_within(got[1].T, {"lse": (want["lse"][0].T, want["lse"][1].T)}, "lse", np.arange(n) != 15)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,k_lens,heads,kv_heads", [([70], [70], 2, 2), ([200], [200], 64, 64), ([256] * 4, [256] * 4, 64, 64), ([53], [2100], 4, 4),
                                                        ([2], [3000], 8, 2)])
def test_lse_of_rows_whose_scores_are_nan(dtype, lens, k_lens, heads, kv_heads):
    """lse is NaN where out is: a row of NaN, and a row that meets NaN in a range of its keys; -inf is left to rows that see nothing."""
    rng = np.random.default_rng(92)
    n, nk = sum(lens), sum(k_lens)
    q, k, v = tensor(rng, dtype, n, heads, 64), tensor(rng, dtype, nk, kv_heads, 64), tensor(rng, dtype, nk, kv_heads, 64)
    plan = layers.AttentionPlan(lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=64, training=False)
    want = R.attention(host(q), host(k), host(v), lens, k_lens, dtype=dtype)["lse"]
    q2 = q.clone()
    q2[1] = NAN
    out, lse = layers.attention(q2, k, v, plan)
    others = np.arange(n) != 1
    assert torch.isnan(out[1]).all() and torch.isnan(lse[:, 1]).all()
    within(lse.T[torch.from_numpy(others).cuda()], (want[0].T[others], want[1].T[others]), "lse")
    k2 = k.clone()
    k2[32:k_lens[0]] = NAN                           # whole tiles, and whole parts where keys are split
    out, lse = layers.attention(q, k2, v, plan)
    assert torch.isnan(out[:lens[0]]).all() and torch.isnan(lse[:, :lens[0]]).all()
    if n > lens[0]:
        within(lse.T[lens[0]:], (want[0].T[lens[0]:], want[1].T[lens[0]:]), "lse")


# sequences of rows and keys, dim, listed positions, size of q and k, of v, of dout
FAR_GRADIENTS = [([2048], [2048], 64, False, 1.0, 1.0, 1e-3), ([2048], [2048], 128, False, 1.0, 1.0, 1e-4), ([1500], [1500], 32, True, 1.0, 1.0, 1e-4),
                 ([64], [20000], 64, False, 1.0, 1.0, 100.0), ([51] * 8, [51] * 8, 32, False, 1.0, 1.0, 1e-5),
                 ([51] * 8, [51] * 8, 64, False, 0.01, 100.0, 3000.0), ([700], [700], 64, False, 0.01, 100.0, 10000.0),
                 ([300], [300], 64, False, 2.0, 3000.0, 0.01), ([300], [300], 64, True, 2.0, 3000.0, 0.01),
                 ([300], [300], 64, False, 2.0, 1.0, 30.0), ([300], [300], 16, False, 2.0, 1.0, 30.0), ([300, 90], [200, 90], 128, False, 2.0, 1.0, 30.0),
                 ([64, 40], [64, 30], 32, False, 2.0, 1.0, 30.0)]


def rounding_of_pairs(q, k, v, dout, out, lens, k_lens, positions, table, buckets):
    """What rounding single pairs to float16 and delta from a rounded out leave in dq, dk and dv, per element, as variances.  A rounding is
    off by at most half a step, 2^-11 of the value, and evenly spread: its variance is at most (2^-11 value)^2 / 3.  delta is off by
    dout . (out - its exact value), known here, and takes that times scale sum_j P_ij k_j from dq."""
    var = {"dq": np.zeros(q.shape), "dk": np.zeros(k.shape), "dv": np.zeros(v.shape)}
    scale, a0, b0 = q.shape[2] ** -0.5, 0, 0
    pos = R.default_positions(lens, k_lens) if positions is None else np.asarray(positions)
    for a, b in zip(lens, k_lens):
        rows, keys = slice(a0, a0 + a), slice(b0, b0 + b)
        for h in range(q.shape[1]):
            Q, K, V, G = q[rows, h], k[keys, h], v[keys, h], dout[rows, h]
            s = scale * Q @ K.T
            if table is not None:
                reach = len(buckets) // 2
                s += table[buckets[np.clip(np.arange(b)[None] - pos[rows][:, None], -reach, reach) + reach], h]
            P = np.exp(s - s.max(1, keepdims=True))
            P /= P.sum(1, keepdims=True)
            y = P @ V
            dS = P * (G @ V.T - (G * y).sum(1, keepdims=True))
            third = 2.0 ** -22 / 3
            off = (G * (out[rows, h] - y)).sum(1, keepdims=True)
            var["dq"][rows, h] = third * scale ** 2 * dS ** 2 @ K ** 2 + (scale * off * (P @ K)) ** 2
            var["dk"][keys, h] = third * scale ** 2 * (dS ** 2).T @ Q ** 2
            var["dv"][keys, h] = third * (P ** 2).T @ G ** 2
        a0, b0 = a0 + a, b0 + b
    return var


@pytest.mark.parametrize("lens,k_lens,dim,given,size,size_v,size_dout", FAR_GRADIENTS)
@pytest.mark.parametrize("biased", [False, True])
def test_float16_gradients_far_from_one(lens, k_lens, dim, given, size, size_v, size_dout, biased):
    """float16 gradients keep their bits where the pairs' own lie below or above what float16 holds: their error's root mean square is that
    of three independent roundings -- the result's, the pairs' and out's (rounding_of_pairs) -- and 4 % for fp32 sums and the sample.
    The bias gradient is summed from dS that is not rounded: the result's alone."""
    rng = np.random.default_rng(93)
    n, nk, heads = sum(lens), sum(k_lens), 2
    q, k, v = tensor(rng, "f16", n, heads, dim, by=size), tensor(rng, "f16", nk, heads, dim, by=size), tensor(rng, "f16", nk, heads, dim, by=size_v)
    dout = tensor(rng, "f16", n, heads, dim, by=size_dout)
    b = table = None
    if biased:
        b, table = layers.relative_buckets(16, 50), tensor(rng, "f16", 16, heads)
    pos = rng.permutation(nk)[:n].astype(np.int32) if given else None
    plan = layers.AttentionPlan(lens, k_lens, heads=heads, head_dim=dim, q_positions=pos)
    out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
    got = layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)
    bias = (None, None) if b is None else (host(table), b.cpu().numpy())
    want = R.attention(host(q), host(k), host(v), lens, k_lens, positions=pos, table=bias[0], buckets=bias[1], dout=host(dout), kernel_out=host(out),
                       dtype="f16")
    var = rounding_of_pairs(host(q), host(k), host(v), host(dout), host(out), lens, k_lens, pos, *bias)
    # where pairs' gradients pass 65504, so do their sums by bucket; rows at listed positions have a test of their own
    for t, name in zip(got, ("dq", "dk", "dv") + (("dtable",) if biased and size_dout < 1000 and not given else ())):
        value = want[name][0]
        assert np.abs(value).max() < 65504, name
        alone = (value.astype(np.float16).astype(np.float64) - value) ** 2
        off = np.sqrt(np.mean((host(t) - value) ** 2))
        most = np.sqrt(np.mean(alone + var.get(name, 0)))
        print(f"{name}: {off / np.sqrt(np.mean(alone)):.3f} times the error of rounding it, {off / most:.3f} of what is left to it")
        assert off <= 1.04 * most, f"{name}: {off / most:.3g} of what is left to it"


def test_tensors_of_forward_mode_differentiation_are_refused():
    """Their tangents would be lost without a word."""
    import torch.autograd.forward_ad as fwad

    rng = np.random.default_rng(94)
    q, k, v = (tensor(rng, "f32", 40, 2, 32) for _ in range(3))
    plan = layers.AttentionPlan([40], heads=2, head_dim=32)
    cos, sin = layers.rotary_table(40, 32)
    gain = torch.ones(32, device="cuda")
    want, _ = layers.attention(q, k, v, plan)
    with fwad.dual_level():
        got, _ = layers.attention(q, k, v, plan)             # nothing to lose
        assert torch.equal(got, want)
        dual = fwad.make_dual(v, torch.ones_like(v))
        with pytest.raises(ValueError, match="tangent"):
            layers.attention(q, k, dual, plan)
        with pytest.raises(ValueError, match="tangent"):
            layers.qk_norm_rope(dual, k, cos, sin)
        with pytest.raises(ValueError, match="tangent"):
            layers.qk_norm_rope(q, k, cos, sin, q_gain=fwad.make_dual(gain, gain))
        with pytest.raises(ValueError, match="tangent"):
            layers.attention_backward(dual, q, k, v, got, torch.zeros(2, 40, device="cuda"), plan)
        with pytest.raises(ValueError, match="tangent"):
            layers.qk_norm_rope_backward(q, dual, q, k, cos, sin)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,keys,heads,dim", [(1500, 1500, 2, 32), (130, 400, 2, 64), (53, 2100, 4, 64), (300, 300, 48, 128)])
def test_bias_gradient_of_listed_positions(dtype, rows, keys, heads, dim):
    """The bias gradient is summed in 32 bits and more from dS that is not rounded, with a delta that owes nothing to the rounding of
    out: what is left is the rounding of the result, and 5 % of it for the fp32 sums and the sample."""
    rng = np.random.default_rng(95)
    q, k, v, dout = tensor(rng, dtype, rows, heads, dim), tensor(rng, dtype, keys, heads, dim), tensor(rng, dtype, keys, heads, dim), tensor(rng, dtype, rows, heads, dim)
    b, table = layers.relative_buckets(16, 50), tensor(rng, dtype, 16, heads)
    pos = rng.permutation(keys)[:rows].astype(np.int32)
    plan = layers.AttentionPlan([rows], [keys], heads=heads, head_dim=dim, q_positions=pos)
    out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
    got = layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)
    want = R.attention(host(q), host(k), host(v), [rows], [keys], positions=pos, table=host(table), buckets=b.cpu().numpy(), dout=host(dout),
                       kernel_out=host(out), dtype=dtype)
    for t, name in zip(got, ("dq", "dk", "dv", "dtable")):
        within(t, want[name], name)
    value = want["dtable"][0]
    rounded = torch.from_numpy(value).to(q.dtype).double().numpy()
    alone, off = (np.sqrt(np.mean((x - value) ** 2)) for x in (rounded, host(got[3])))
    print(f"dtable: {off / alone:.3f} times the error of rounding it")
    assert off <= 1.05 * alone


# five sequences of 64 heads fill the card: tiles of 128 rows in the forward kernel, four wavefronts in both backward ones; fewer heads take
# tiles of 64 and two wavefronts
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("buckets", [None, (16, 50, True)])
@pytest.mark.parametrize("heads,kinds", [(64, (0, 4, 4)), (20, (1, 2, 2))])
def test_kernels_that_large_batches_take(dtype, dim, buckets, heads, kinds):
    """The plan says which kernels ran; rows in order, ragged lengths, a window with first tokens."""
    plan = attend(dtype, dim, [256, 250, 199, 128, 1], heads=heads, kv_heads=heads, window=(90, 40), sinks=2, buckets=buckets, seed=97, packed=True)
    assert tuple(int(x) for x in plan.words[[11, 19, 22]]) == kinds


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_kernels_that_large_batches_take_with_shared_heads(dtype, dim):
    plan = attend(dtype, dim, [256] * 4, heads=128, kv_heads=64, window=(-1, 0), buckets=(16, 50, False), seed=98)
    assert tuple(int(x) for x in plan.words[[11, 19, 22]]) == (0, 4, 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,heads,kinds", [([256, 250, 199, 128, 1], 64, (0, 4, 4)), ([200, 190], 40, (1, 2, 2))])
def test_hidden_places_in_the_kernels_that_large_batches_take(dtype, lens, heads, kinds):
    """Keys, values, queries and gradients of NaN and infinity reach what sees them and nothing else."""
    rng = np.random.default_rng(99)
    n, window = sum(lens), (9, 4)
    q, k, v, dout = (tensor(rng, dtype, n, heads, 64) for _ in range(4))
    plan = layers.AttentionPlan(lens, heads=heads, head_dim=64, window=window)
    assert tuple(int(x) for x in plan.words[[11, 19, 22]]) == kinds
    out, lse = layers.attention(q, k, v, plan)
    want = R.attention(host(q), host(k), host(v), lens, lens, window, dout=host(dout), kernel_out=host(out), dtype=dtype)
    start = np.repeat(np.cumsum([0] + lens[:-1]), lens)
    p, j = np.arange(n)[:, None], np.arange(n)[None]
    see = (j <= p + window[1]) & (j >= p - window[0]) & (start[:, None] == start[None])
    # keys and values; 140 and 131 lie in a tile with rows that do not see them
    k2, v2 = k.clone(), v.clone()
    k2[140], v2[131, :, 3] = NAN, INF
    out2, lse2 = layers.attention(q, k2, v2, plan)
    dq, dk, dv, _ = layers.attention_backward(dout, q, k2, v2, out2, lse2, plan)
    met = see[:, [140, 131]].any(1)
    for t, name in ((out2, "out"), (dq, "dq")):
        rows_within(t, want, name, ~met)
        assert not np.isfinite(host(t)[met]).all(axis=(1, 2)).any()
    rows_within(lse2.T, {"lse": (want["lse"][0].T, want["lse"][1].T)}, "lse", ~see[:, 140])
    rows_within(dk, want, "dk", ~see[met].any(0))
    rows_within(dv, want, "dv", ~see[see[:, 140]].any(0))
    # a row
    q2, dout2 = q.clone(), dout.clone()
    q2[150], dout2[150] = NAN, INF
    out3, lse3 = layers.attention(q2, k, v, plan)
    dq, dk, dv, _ = layers.attention_backward(dout2, q2, k, v, out3, lse3, plan)
    rows_within(out3, want, "out", np.arange(n) != 150)
    rows_within(dq, want, "dq", np.arange(n) != 150)
    for t, name in ((dk, "dk"), (dv, "dv")):
        rows_within(t, want, name, ~see[150])
        assert not np.isfinite(host(t)[see[150]]).any()


def test_kernels_that_large_batches_take_with_the_most_shared_memory():
    """fp32 heads of 128 with the largest bias and four wavefronts in both backward kernels, rows in order."""
    plan = attend("f32", 128, [256] * 4, heads=64, kv_heads=64, window=(200, 100), buckets=(64, 1024, True), seed=100)
    assert tuple(int(x) for x in plan.words[[11, 19, 22]]) == (0, 4, 4)
