"""Layer operators (deepptmpred_amd/layers.py) on the GPU against their restatement in float64 (oracle/layers_ref.py), whose
bounds follow the kernels' roundings: every element of every output has to be within its own bound."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from deepptmpred_amd import _native, layers, spec  # noqa: E402
from oracle import layers_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def tensor(rng, dtype, *shape, by=1.0):
    return torch.from_numpy(rng.normal(0, by, shape).astype(np.float32)).to(TYPES[dtype]).cuda()


def host(t):
    return t.detach().cpu().double().numpy()


def within(got, want, what):
    value, bound = want
    got = host(got)
    assert got.shape == value.shape, what
    both = np.isfinite(value)
    assert np.array_equal(np.isfinite(got), both) and np.array_equal(got[~both & ~np.isnan(value)], value[~both & ~np.isnan(value)]), what
    off = np.abs(got - value)[both] / np.maximum(bound[both], 1e-300)
    assert off.size == 0 or off.max() <= 1.0, f"{what}: {off.max():.3g} of its bound"


def attend(dtype, dim, q_lens, k_lens=None, heads=2, kv_heads=2, window=(-1, -1), sinks=0, buckets=None, positions=None,
           train=True, seed=0, scale=None, packed=False):
    rng = np.random.default_rng(seed)
    k_lens = q_lens if k_lens is None else k_lens
    nq, nk = sum(q_lens), sum(k_lens)
    if packed:
        x = tensor(rng, dtype, nq, heads + 2 * kv_heads, dim)
        q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    else:
        q, k, v = tensor(rng, dtype, nq, heads, dim), tensor(rng, dtype, nk, kv_heads, dim), tensor(rng, dtype, nk, kv_heads, dim)
    table = b = None
    if buckets:
        b = layers.relative_buckets(*buckets)
        table = tensor(rng, dtype, buckets[0], heads, by=0.7)
    plan = layers.AttentionPlan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=dim, window=window, sinks=sinks,
                                q_positions=positions, training=train)
    out, lse = layers.attention(q, k, v, plan, scale=scale, table=table, buckets=b)
    dout = tensor(rng, dtype, nq, heads, dim) if train else None
    got = {"out": out, "lse": lse}
    if train:
        got["dq"], got["dk"], got["dv"], dt = layers.attention_backward(dout, q, k, v, out, lse, plan, scale=scale, table=table, buckets=b)
        if buckets:
            got["dtable"] = dt
    want = R.attention(host(q), host(k), host(v), q_lens, k_lens, window, sinks, positions, scale,
                       None if table is None else host(table), None if b is None else b.cpu().numpy(),
                       None if dout is None else host(dout), host(out), dtype)
    for n in got:
        within(got[n], want[n], n)
    return plan


LENGTHS = {"one": [1], "odd": [51, 7, 64], "ragged": [0, 33, 1, 130, 65, 0], "long": [300]}
MASKS = {"full": ((-1, -1), 0), "back": ((-1, 0), 0), "window": ((20, 13), 3), "self": ((0, 0), 1), "ahead": ((5, -1), 2)}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_attention_lengths(dtype, dim, lengths):
    attend(dtype, dim, LENGTHS[lengths], seed=dim)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("buckets", [None, (32, 40, True), (8, 1000, True), (8, 9, False)])
def test_attention_masks_and_bias(dtype, mask, buckets):
    window, sinks = MASKS[mask]
    attend(dtype, 32, [150, 70, 3], heads=4, kv_heads=2, window=window, sinks=sinks, buckets=buckets, seed=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,lengths,mode", [(64, 64, [40] * 5, 1), (48, 16, [129] * 6, 0), (40, 40, [200, 51, 128, 300, 257, 120], 0)])
@pytest.mark.parametrize("buckets", [None, (16, 50, True)])
def test_attention_tiles_of_many_rows(dtype, heads, kv_heads, lengths, mode, buckets):
    """Batches large enough for the kernels that share tiles of keys between wavefronts."""
    plan = attend(dtype, 64, lengths, heads=heads, kv_heads=kv_heads, window=(90, 40), sinks=2, buckets=buckets, seed=5, packed=True)
    assert plan.words[11] in (mode, 0, 1)


@pytest.mark.parametrize("dim", [16, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_tiles_of_many_rows_other_dims(dtype, dim):
    attend(dtype, dim, [100] * 6, heads=48, kv_heads=48, window=(-1, 0), seed=6)
    attend(dtype, dim, [140] * 6, heads=48, kv_heads=24, window=(33, 20), sinks=1, buckets=(16, 30, True), seed=7)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_attention_few_queries(dtype, dim):
    """One new token behind caches (one of them empty), and the sites of proteins in any order, the keys split over
    wavefronts and workgroups."""
    attend(dtype, dim, [1] * 5, [700, 0, 1, 33, 1500], heads=8, kv_heads=2, window=(600, 0), sinks=4, train=False, seed=8)
    rng = np.random.default_rng(9)
    pos = np.concatenate([rng.permutation(2100)[:53], rng.permutation(480)[:36]]).astype(np.int32)
    attend(dtype, dim, [53, 36], [2100, 480], heads=4, kv_heads=4, positions=pos, buckets=(32, 128, True), seed=10)
    attend(dtype, dim, [53, 36], [2100, 480], heads=4, kv_heads=1, positions=pos, window=(100, 60), sinks=5, seed=11)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_heads_that_share_keys_share_a_tile(dtype):
    attend(dtype, 32, [3, 1, 4], [400, 65, 4], heads=24, kv_heads=4, window=(300, 0), buckets=(32, 128, False), sinks=2, seed=30)
    attend(dtype, 64, [1], [900], heads=16, kv_heads=2, buckets=(64, 1000, False), window=(-1, 0), train=False, seed=31)
    attend(dtype, 64, [20, 13], [90, 40], heads=12, kv_heads=4, buckets=(16, 50, True), seed=32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_given_positions_in_training(dtype):
    """Rows at positions from a list, in any order, in the kernels of large batches too: bias gradient and masks."""
    rng = np.random.default_rng(33)
    lens = [140] * 6
    pos = np.concatenate([rng.permutation(200)[:140] - 20 for _ in lens]).astype(np.int32)
    attend(dtype, 32, lens, heads=48, kv_heads=24, positions=pos, window=(60, 50), sinks=3, buckets=(32, 40, True), seed=34)
    attend(dtype, 64, [70], [90], heads=2, kv_heads=1, positions=rng.permutation(90)[:70].astype(np.int32), buckets=(8, 9, True), seed=35)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_rows_that_see_nothing(dtype):
    """More queries than keys under a window that only looks back: the first stand before the first key; positions far off;
    sequences without keys or without queries."""
    attend(dtype, 64, [40, 5, 0, 3], [10, 0, 7, 3], window=(4, 0), seed=12)
    attend(dtype, 64, [6], [100], window=(3, 3), positions=np.array([-500, -4, 0, 99, 104, 5000], np.int32), seed=13)


def test_bias_that_hides():
    """Table entries of -inf or the type's lowest value hide their pairs; a row whose pairs are all hidden is empty."""
    rng = np.random.default_rng(14)
    for low in (-np.inf, float(torch.finfo(torch.bfloat16).min)):
        q, k, v, dout = (tensor(rng, "bf16", 70, 2, 32) for _ in range(4))
        b = layers.relative_buckets(8, 9, True)
        table = tensor(rng, "bf16", 8, 2)
        table[3:, 0] = low          # of head 0 only three distances stay
        table[:, 1] = low
        plan = layers.AttentionPlan([70], heads=2, head_dim=32)
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        assert not out[:, 1].any() and torch.isneginf(lse[1]).all()
        grads = layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)
        want = R.attention(host(q), host(k), host(v), [70], [70], table=host(table), buckets=b.cpu().numpy(), dout=host(dout),
                           kernel_out=host(out), dtype="bf16")
        for n, t in zip(("out", "lse", "dq", "dk", "dv", "dtable"), (out, lse) + grads):
            within(t, want[n], n)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [200, 40])
def test_what_hidden_places_hold_does_not_matter(dtype, rows):
    """Keys and values of NaN and infinity reach the rows that see them and no other, in both directions."""
    rng = np.random.default_rng(15)
    heads = 48 if rows == 200 else 2
    q, k, v, dout = (tensor(rng, dtype, rows, heads, 64) for _ in range(4))
    plan = layers.AttentionPlan([rows], heads=heads, head_dim=64, window=(9, 4))
    out, lse = layers.attention(q, k, v, plan)
    grads = layers.attention_backward(dout, q, k, v, out, lse, plan)
    k2, v2, q2, dout2 = k.clone(), v.clone(), q.clone(), dout.clone()
    k2[20], v2[20], v2[21, :, 3] = float("nan"), float("nan"), float("inf")
    out2, lse2 = layers.attention(q, k2, v2, plan)
    sees = torch.zeros(rows, dtype=torch.bool, device="cuda")
    sees[16:30] = True              # rows with 20 in [p - 9, p + 4]
    clear = ~sees
    clear[17:31] = False            # and those of 21
    want = R.attention(host(q), host(k), host(v), [rows], [rows], (9, 4), dout=host(dout), kernel_out=host(out), dtype=dtype)

    def near(t, name, keep):
        value, bound = want[name]
        k = keep.cpu().numpy()
        value, bound = (value[:, k], bound[:, k]) if name == "lse" else (value[k], bound[k])
        within(t[:, keep] if name == "lse" else t[keep], (value, bound), name)

    near(out2, "out", clear)
    near(lse2, "lse", clear)
    assert torch.isnan(out2[sees]).all()
    assert torch.isposinf(out2[30, :, 3]).all() and torch.isfinite(out2[30, :, :3]).all()
    # a row whose query and gradient are not finite reaches the keys it sees alone
    r = 100 % rows
    q2[r], dout2[r] = float("nan"), float("inf")
    out3, lse3 = layers.attention(q2, k, v, plan)
    grads3 = layers.attention_backward(dout2, q2, k, v, out3, lse3, plan)
    keys = torch.zeros(rows, dtype=torch.bool, device="cuda")
    keys[max(0, r - 9):r + 5] = True
    near(grads3[0], "dq", torch.arange(rows, device="cuda") != r)
    for t, name in zip(grads3[1:3], ("dk", "dv")):
        near(t, name, ~keys)
        assert not torch.isfinite(t[keys]).any()
    # and keys that are not finite leave the gradients of the rows that do not see them
    grads4 = layers.attention_backward(dout, q, k2, v2, out2, lse2, plan)
    near(grads4[0], "dq", clear)
    assert torch.isnan(grads4[0][sees]).all()


def test_strides_and_rows_behind_the_last():
    """Head-major tensors, broadcast rows and heads, results written into views; what lies behind a sequence stays."""
    rng = np.random.default_rng(16)
    lens, heads, dim = [37, 90], 4, 64
    n = sum(lens)
    plan = layers.AttentionPlan(lens, heads=heads, kv_heads=heads, head_dim=dim)
    q, k, v, dout = (tensor(rng, "bf16", n, heads, dim) for _ in range(4))
    out, lse = layers.attention(q, k, v, plan)
    grads = layers.attention_backward(dout, q, k, v, out, lse, plan)

    def major(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def longer(t):
        return torch.cat([t, torch.full_like(t[:5], float("nan"))])

    wide = torch.full((n + 5, 3 * heads, dim), 7.0, dtype=q.dtype, device="cuda")
    out2, lse2 = layers.attention(longer(major(q)), longer(k), major(v), plan, out=wide[:, heads:2 * heads])
    assert torch.equal(wide[:n, heads:2 * heads], out) and torch.equal(lse2, lse)
    assert (wide[n:] == 7).all() and (wide[:, :heads] == 7).all() and (wide[:, 2 * heads:] == 7).all()
    gw = torch.full((n + 5, 3 * heads, dim), 7.0, dtype=q.dtype, device="cuda")
    layers.attention_backward(longer(dout), major(q), longer(k), v, longer(out), lse, plan, dq=gw[:, :heads],
                              dk=gw[:, heads:2 * heads], dv=gw[:, 2 * heads:])
    assert torch.equal(gw[:n], torch.cat(grads[:3], 1)) and (gw[n:] == 7).all()
    # one head for all, one row for all
    k1, v1 = k[:, :1].expand(n, heads, dim), v[:1].expand(n, heads, dim)
    a, la = layers.attention(q, k1, v1, plan)
    b, lb = layers.attention(q, k1.contiguous(), v1.contiguous(), plan)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_equal_calls_give_equal_bits_on_any_stream():
    rng = np.random.default_rng(17)
    lens = [300, 1, 77, 512]
    q, k, v, dout = (tensor(rng, "bf16", sum(lens), 4, 64) for _ in range(4))
    b = layers.relative_buckets(32, 128)
    table = tensor(rng, "bf16", 32, 4)
    plan = layers.AttentionPlan(lens, heads=4, head_dim=64, window=(100, 100), sinks=2)

    def run():
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        return (out, lse) + layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))


def test_captured_graphs():
    """Two graphs recorded from the same tensors, replayed in turn with eager work between, leave the eager results."""
    rng = np.random.default_rng(18)
    lens = [200, 33, 480]
    x = tensor(rng, "bf16", sum(lens), 12, 64)
    dout = tensor(rng, "bf16", sum(lens), 4, 64)
    cos, sin = layers.rotary_table(512, 64)
    gain = torch.ones(64, device="cuda")
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    plan = layers.AttentionPlan(lens, heads=4, head_dim=64, window=(64, 64), sinks=1)
    table, b = tensor(rng, "bf16", 32, 4), layers.relative_buckets(32, 128)

    def run():
        q, k = layers.qk_norm_rope(x[:, :4], x[:, 4:8], cos, sin, q_gain=gain, k_gain=gain, positions=pos)
        out, lse = layers.attention(q, k, x[:, 8:], plan, table=table, buckets=b)
        dq, dk, dv, dt = layers.attention_backward(dout, q, k, x[:, 8:], out, lse, plan, table=table, buckets=b)
        return (out, lse, dv, dt) + layers.qk_norm_rope_backward(dq, dk, x[:, :4], x[:, 4:8], cos, sin, q_gain=gain, k_gain=gain, positions=pos)

    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = run()
        graphs.append((g, r))
    for step in range(3):
        x.copy_(tensor(np.random.default_rng(100 + step), "bf16", *x.shape))
        want = run()
        for g, r in graphs:
            for t in r:
                t.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(r, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 1, 1), (77, 3, 1), (515, 20, 20)])
def test_norm_and_rotation(dtype, dim, interleaved, rows, heads, kv_heads):
    rng = np.random.default_rng(dim + rows)
    x = tensor(rng, dtype, rows, heads + 2 * kv_heads, dim, by=1.5)
    q, k = x[:, :heads], x[:, heads:heads + kv_heads]
    dq2, dk2 = tensor(rng, dtype, rows, heads, dim), tensor(rng, dtype, rows, kv_heads, dim)
    gq, gk = (torch.from_numpy(rng.normal(1, 0.3, dim).astype(np.float32)).cuda() for _ in range(2))
    cos, sin = layers.rotary_table(20011, dim)
    pos = torch.from_numpy(rng.integers(0, 20011, rows).astype(np.int32)).cuda()
    p = pos.cpu().numpy()
    for a, b in ((gq, gk), (None, gk), (None, None)):
        more = dict(q_gain=a, k_gain=b, positions=pos, interleaved=interleaved)
        y = layers.qk_norm_rope(q, k, cos, sin, **more)
        g = layers.qk_norm_rope_backward(dq2, dk2, q, k, cos, sin, **more)
        for t, gain, dy, i in ((q, a, dq2, 0), (k, b, dk2, 1)):
            want = R.qk_norm_rope(host(t), None if gain is None else host(gain), host(cos), host(sin), p, 1e-6, interleaved, host(dy), dtype)
            within(y[i], want["y"], f"y{i}")
            within(g[i], want["dx"], f"dx{i}")
            if gain is None:
                assert g[2 + i] is None
            else:
                within(g[2 + i], want["dgain"], f"dgain{i}")


def test_norm_and_rotation_in_place_default_positions_and_bad_ones():
    rng = np.random.default_rng(21)
    cos, sin = layers.rotary_table(64, 64)
    gain = torch.full((64,), 1.1, device="cuda")
    x = tensor(rng, "bf16", 64, 9, 64)
    q, k = layers.qk_norm_rope(x[:, :4], x[:, 4:6], cos, sin, q_gain=gain, k_gain=gain)
    pos = torch.arange(64, device="cuda", dtype=torch.int32)
    q2, k2 = layers.qk_norm_rope(x[:, :4], x[:, 4:6], cos, sin, q_gain=gain, k_gain=gain, positions=pos)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    y = x.clone()
    layers.qk_norm_rope(y[:, :4], y[:, 4:6], cos, sin, q_gain=gain, k_gain=gain, q_out=y[:, :4], k_out=y[:, 4:6])
    assert torch.equal(y[:, :4], q) and torch.equal(y[:, 4:6], k) and torch.equal(y[:, 6:], x[:, 6:])
    pos[5], pos[9] = 64, -1
    q3, k3 = layers.qk_norm_rope(x[:, :4], x[:, 4:6], cos, sin, q_gain=gain, k_gain=gain, positions=pos)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[[5, 9]] = True
    assert torch.isnan(q3[bad]).all() and torch.isnan(k3[bad]).all() and torch.equal(q3[~bad], q[~bad])
    e = x[:0]
    q4, k4 = layers.qk_norm_rope(e[:, :4], e[:, 4:6], cos, sin, q_gain=gain, k_gain=gain)
    assert q4.shape == (0, 4, 64) and k4.shape == (0, 2, 64)
    g = layers.qk_norm_rope_backward(e[:, :4], e[:, 4:6], e[:, :4], e[:, 4:6], cos, sin, q_gain=gain, k_gain=gain)
    assert not g[2].any() and not g[3].any()


def test_empty_batches():
    e = torch.empty(0, 2, 64, device="cuda")
    for lens in ([], [0, 0]):
        plan = layers.AttentionPlan(lens, heads=2, head_dim=64)
        out, lse = layers.attention(e, e, e, plan)
        assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
        b = layers.relative_buckets(8, 9)
        dq, dk, dv, dt = layers.attention_backward(e, e, e, e, out, lse, plan, table=torch.ones(8, 2, device="cuda"), buckets=b)
        assert dq.shape == (0, 2, 64) and not dt.any()


def test_gradients_against_differences():
    """Every gradient along a random direction against the central difference of the float64 forward pass."""
    rng = np.random.default_rng(22)
    lens, heads, dim = [30, 45], 2, 32
    x = {n: rng.normal(0, 1, (75, heads, dim)) for n in "qkv"}
    x["t"] = rng.normal(0, 0.7, (8, heads))
    x = {n: a.astype(np.float32).astype(np.float64) for n, a in x.items()}
    w = rng.normal(0, 1, (75, heads, dim)).astype(np.float32)
    b = layers.relative_buckets(8, 9)
    dev = {n: torch.from_numpy(a.astype(np.float32)).cuda() for n, a in x.items()}
    plan = layers.AttentionPlan(lens, heads=heads, head_dim=dim, window=(20, 6), sinks=2)
    out, lse = layers.attention(dev["q"], dev["k"], dev["v"], plan, table=dev["t"], buckets=b)
    grads = layers.attention_backward(torch.from_numpy(w).cuda(), dev["q"], dev["k"], dev["v"], out, lse, plan, table=dev["t"], buckets=b)

    def loss(y):
        r = R.attention(y["q"], y["k"], y["v"], lens, lens, (20, 6), 2, table=y["t"], buckets=b.cpu().numpy())
        return float((r["out"][0] * w).sum())

    step = 1e-5
    for n, g in zip("qkvt", grads):
        d = rng.normal(0, 1, x[n].shape)
        up, down = dict(x), dict(x)
        up[n], down[n] = x[n] + step * d, x[n] - step * d
        slope = (loss(up) - loss(down)) / (2 * step)
        # the difference is off by O(step^2) and 64-bit rounding / step; the kernel by fp32 sums
        assert abs(float((host(g) * d).sum()) - slope) <= 1e-4 * (1 + float(np.abs(host(g) * d).sum()) / 10), n


def test_a_layer_in_front_of_the_classifier():
    """The operators in a row, as a residue encoder's layer runs them -- norm and rotation, attention with bias -- whose
    1280-wide rows the classifier then scores on the device, and only the site rows of the same layer scored the same way."""
    rng = np.random.default_rng(23)
    L, heads, dim = 300, 20, 64
    x = tensor(rng, "f32", L, 3 * heads, dim)
    gq, gk = torch.ones(dim, device="cuda"), torch.ones(dim, device="cuda")
    cos, sin = layers.rotary_table(1024, dim)
    b = layers.relative_buckets(32, 128)
    table = tensor(rng, "f32", 32, heads, by=0.5)
    q, k = layers.qk_norm_rope(x[:, :heads], x[:, heads:2 * heads], cos, sin, q_gain=gq, k_gain=gk)
    v = x[:, 2 * heads:]
    plan = layers.AttentionPlan([L], heads=heads, head_dim=dim)
    out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
    p = np.arange(L)
    hq = R.qk_norm_rope(host(x[:, :heads]), host(gq), host(cos), host(sin), p)["y"][0]
    hk = R.qk_norm_rope(host(x[:, heads:2 * heads]), host(gk), host(cos), host(sin), p)["y"][0]
    want = R.attention(hq, hk, host(v), [L], [L], table=host(table), buckets=b.cpu().numpy())["out"][0]
    # q and k carry their own rounding into the scores: (D + 12) U of |q|.|k| scale, doubled by the softmax
    assert np.abs(host(out) - want).max() <= 1e-4
    sites = np.sort(rng.permutation(L)[:53]).astype(np.int32)
    few = layers.AttentionPlan([len(sites)], [L], heads=heads, head_dim=dim, q_positions=sites, training=False)
    rows, _ = layers.attention(q[torch.from_numpy(sites).long().cuda()].contiguous(), k, v, few, table=table, buckets=b)
    assert float((rows - out[torch.from_numpy(sites).long().cuda()]).abs().max()) <= 1e-5

    # the scorer's NULL stream is its own: the rows are handed over on a stream that both sides name
    scorer = _native.Scorer(spec.pack_blob(spec.synthetic_weights(7)), spec.DEFAULT_SPEC, 0)
    codes = rng.integers(0, 20, L).astype(np.uint8)
    strct = rng.normal(0, 1, (53, 8)).astype(np.float32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        c, st, at = torch.from_numpy(codes).cuda(), torch.from_numpy(strct).cuda(), torch.from_numpy(sites + 1).cuda()
        proba = torch.empty(53, 2, device="cuda")
        again, _ = layers.attention(q, k, v, plan, table=table, buckets=b)
        scorer.score_protein_device(c.data_ptr(), L, again.data_ptr(), L, at.data_ptr(), st.data_ptr(), 53, proba.data_ptr(),
                                    stream.cuda_stream)
    stream.synchronize()
    want = scorer.score_protein(codes, out.reshape(L, 1280).cpu().numpy(), sites + 1, strct)
    assert np.abs(proba.cpu().numpy() - want).max() <= 1e-6
    scorer.close()


@pytest.mark.parametrize("given", [False, True])
def test_most_shared_memory(given):
    """fp32 heads of 128 with the largest bias: four wavefronts of the backward pass, and eight heads in a tile."""
    rng = np.random.default_rng(40)
    pos = rng.permutation(1024).astype(np.int32) if given else None
    attend("f32", 128, [1024] if given else [256] * 2, [1500] if given else None, heads=64, kv_heads=64, positions=pos, window=(200, 100),
           buckets=(64, 1024, True), seed=41)
    attend("f32", 128, [3, 4], [1300, 40], heads=16, kv_heads=2, buckets=(64, 1024, False), train=False, seed=42)


def test_a_plan_dropped_while_another_stream_reads_it():
    """The plan's memory is not handed out again before the calls that read it have run."""
    rng = np.random.default_rng(43)
    q, k, v = (tensor(rng, "bf16", 900, 2, 64) for _ in range(3))
    want, _ = layers.attention(q, k, v, layers.AttentionPlan([900], heads=2, head_dim=64))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = layers.AttentionPlan([900], heads=2, head_dim=64)
    at, size = plan.device_words.data_ptr(), plan.device_words.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(2e8))                 # some 0.1 s
        out, _ = layers.attention(q, k, v, plan)
    del plan
    new = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not side.query() and all(t.data_ptr() != at for t in new)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 64])
@pytest.mark.parametrize("buckets", [None, (32, 40, True), (8, 9, False), (8, 200, True)])
def test_short_sequences(dtype, dim, buckets):
    """Windows: dq, dk, dv and the bias gradient from one kernel.  Sequences without rows or keys, of one, of a wavefront's 32, of
    all 64; rows in front of the first key and keys that no row sees."""
    attend(dtype, dim, [51, 64, 33, 1, 21, 32], heads=3, kv_heads=3, buckets=buckets, seed=50, packed=True)
    attend(dtype, dim, [0, 3, 64, 0, 10, 1, 40], [5, 64, 3, 0, 0, 1, 33], buckets=buckets, window=(20, 13), sinks=3, seed=51)
    attend(dtype, dim, [64, 64], [64, 2], heads=1, kv_heads=1, buckets=buckets, window=(-1, 0), seed=52)
    attend(dtype, dim, [21, 32, 0, 7, 1], [21, 32, 3, 0, 30], heads=3, kv_heads=3, buckets=buckets, window=(12, 9), sinks=1, seed=54)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [51, 32])
def test_short_sequences_with_hidden_nan(dtype, rows):
    """What a hidden key or row of a window holds does not reach the gradients of the others, and rows behind stay as they are."""
    rng = np.random.default_rng(53)
    lens, n = [rows, rows - 8], 2 * rows - 8
    last = rows - 1
    q, k, v, dout = (tensor(rng, dtype, n, 2, 32) for _ in range(4))
    plan = layers.AttentionPlan(lens, heads=2, head_dim=32, window=(-1, 0))
    b = layers.relative_buckets(8, 20)
    table = tensor(rng, dtype, 8, 2)

    def run(q, k, v, dout):
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        into = {x: torch.full((n + 2, 2, 32), 7.0, dtype=q.dtype, device="cuda") for x in ("dq", "dk", "dv")}
        layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b, **into)
        assert all((x[n:] == 7.0).all() for x in into.values())
        return out, [x[:n] for x in into.values()]

    out, plain = run(q, k, v, dout)
    want = R.attention(host(q), host(k), host(v), lens, lens, (-1, 0), 0, None, None, host(table), b.cpu().numpy(), host(dout), host(out), dtype)

    def near(t, name, rows):
        within(t[rows], (want[name][0][rows], want[name][1][rows]), name)

    for t, name in zip(plain, ("dq", "dk", "dv")):
        near(t, name, slice(0, n))
    k2, v2 = k.clone(), v.clone()
    k2[last], v2[last] = float("nan"), float("inf")       # seen by the last row alone
    out2, (dq, _, _) = run(q, k2, v2, dout)
    near(dq, "dq", slice(0, last))
    near(dq, "dq", slice(rows, n))
    assert torch.isfinite(out2[:last]).all() and not torch.isfinite(out2[last]).any()
    q2, dout2 = q.clone(), dout.clone()
    q2[0], dout2[0] = float("nan"), float("inf")      # sees key 0 alone
    _, (_, dk, dv) = run(q2, k, v, dout2)
    for t, name in ((dk, "dk"), (dv, "dv")):
        near(t, name, slice(1, n))
        assert not torch.isfinite(t[0]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("buckets", [None, (16, 50, True)])
def test_keys_that_no_row_sees(dtype, buckets):
    """Sequences without rows, and keys ahead of every row: zeros in dk and dv, nothing in the bias gradient."""
    attend(dtype, 64, [0, 200, 30], [130, 200, 400], heads=4, kv_heads=2, buckets=buckets, window=(60, 0), seed=60)
    pos = np.arange(90, dtype=np.int32)
    attend(dtype, 64, [90], [500], heads=4, kv_heads=4, positions=pos, buckets=buckets, window=(40, 5), seed=61)


def test_offsets_past_32_bits():
    """Rows 16 MiB apart: 300 of them span 4.7 GB, forward and backward, rows and keys."""
    rng = np.random.default_rng(62)
    n, heads, dim, row = 300, 2, 64, 1 << 23                  # elements of two bytes between rows
    buf = torch.empty(n * row, dtype=torch.bfloat16, device="cuda")
    at = iter(range(0, 1 << 20, 4096))

    def far(x=None):
        t = buf.as_strided((n, heads, dim), (row, dim, 1), next(at))
        return t if x is None else t.copy_(x)

    q, k, v, dout = (tensor(rng, "bf16", n, heads, dim) for _ in range(4))
    plan = layers.AttentionPlan([n], heads=heads, head_dim=dim, window=(150, 100))
    cos, sin = layers.rotary_table(n, dim)
    gain = torch.ones(dim, device="cuda")

    def run(f):
        a, b, c, g = f(q), f(k), f(v), f(dout)
        a, b = layers.qk_norm_rope(a, b, cos, sin, q_gain=gain, k_gain=gain, q_out=f(), k_out=f())
        out, lse = layers.attention(a, b, c, plan, out=f())
        dq, dk, dv, _ = layers.attention_backward(g, a, b, c, out, lse, plan, dq=f(), dk=f(), dv=f())
        return [t.clone() for t in (a, b, out, lse, dq, dk, dv)]

    near = run(lambda x=None: torch.empty(n, heads, dim, dtype=torch.bfloat16, device="cuda") if x is None else x.clone())
    for x, y in zip(run(far), near):
        assert torch.equal(x, y)


def test_captured_with_the_most_shared_memory():
    """Kernels that need more than 64 KB of it are set up outside the stream: a first call may be a captured one."""
    rng = np.random.default_rng(63)
    q, k, v, dout = (tensor(rng, "f32", 256, 48, 128) for _ in range(4))
    b = layers.relative_buckets(64, 900)
    table = tensor(rng, "f32", 64, 48)
    plan = layers.AttentionPlan([256], heads=48, head_dim=128, window=(90, 90))

    def run():
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        return (out, lse) + layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = run()
    for step in range(3):
        q.copy_(tensor(np.random.default_rng(70 + step), "f32", *q.shape))
        for t in r:
            t.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(r, run()))


def test_an_error_of_an_earlier_call_is_not_reported_again():
    """A call refused for its device leaves the next one alone."""
    lib = _native.load_library()
    rng = np.random.default_rng(80)
    q, k, v = (tensor(rng, "bf16", 70, 2, 64) for _ in range(3))
    plan = layers.AttentionPlan([70], heads=2, head_dim=64)
    want, _ = layers.attention(q, k, v, plan)
    rows = [_native.Rows(t.data_ptr(), 70, 128, 64) for t in (q, k, v, torch.empty_like(q))]
    x = _native.AttentionArgs(plan=plan.words.ctypes.data, plan_dev=plan.device_words.data_ptr(), q=rows[0], k=rows[1], v=rows[2], out=rows[3],
                              lse=torch.empty(140, device="cuda").data_ptr(), dtype=_native.PRECISIONS["bf16"], device=4096, scale=0.125)
    assert lib.dptm_attention_forward(C.addressof(x)) == _native.DPTM_EINVAL and b"no such device" in lib.dptm_layer_last_error()
    got, _ = layers.attention(q, k, v, plan)
    assert torch.equal(got, want)


def test_norm_and_rotation_backward_in_place():
    """Gradients in the place of the ones they are made from, or of the rows; a gain for one of the two tensors only."""
    rng = np.random.default_rng(81)
    cos, sin = layers.rotary_table(200, 64)
    gain = torch.full((64,), 0.9, device="cuda")
    x, g = tensor(rng, "bf16", 200, 6, 64), tensor(rng, "bf16", 200, 6, 64)
    for gains in ({"q_gain": gain, "k_gain": gain}, {"q_gain": gain}, {"k_gain": gain}, {}):
        want = layers.qk_norm_rope_backward(g[:, :4], g[:, 4:], x[:, :4], x[:, 4:], cos, sin, **gains)
        g2, x2 = g.clone(), x.clone()
        got = layers.qk_norm_rope_backward(g2[:, :4], g2[:, 4:], x[:, :4], x[:, 4:], cos, sin, dq=g2[:, :4], dk=g2[:, 4:], **gains)
        into = layers.qk_norm_rope_backward(g[:, :4], g[:, 4:], x2[:, :4], x2[:, 4:], cos, sin, dq=x2[:, :4], dk=x2[:, 4:], **gains)
        for a, b, c, name in zip(want, got, into, ("q_gain", "k_gain", "q_gain", "k_gain")):
            assert (a is None and b is None and c is None) or (torch.equal(a, b) and torch.equal(a, c)), name
        assert (want[2] is None) == ("q_gain" not in gains) and (want[3] is None) == ("k_gain" not in gains)


def test_two_threads_at_once():
    """Calls of two host threads, each on a stream of its own."""
    import threading

    rng = np.random.default_rng(82)
    b = layers.relative_buckets(16, 50)
    jobs = []
    for n, heads, dim in ((300, 4, 64), (70, 2, 32)):
        t = [tensor(rng, "bf16", n, heads, dim) for _ in range(4)]
        jobs.append((t, layers.AttentionPlan([n], heads=heads, head_dim=dim), tensor(rng, "bf16", 16, heads)))

    def run(job):
        (q, k, v, dout), plan, table = job
        out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
        return (out, lse) + layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                r = run(jobs[i])
            s.synchronize()
            if not all(torch.equal(a, c) for a, c in zip(r, want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[51, 17, 64], [21, 32]])
def test_short_sequences_in_packed_tensors(dtype, lens):
    """Inputs and gradients as columns of packed tensors, [rows][heads][q k v][dim] too; the columns between are left alone."""
    rng = np.random.default_rng(83)
    n = sum(lens)
    plan = layers.AttentionPlan(lens, heads=3, head_dim=32, window=(30, 10), sinks=1)
    b = layers.relative_buckets(16, 20)
    table = tensor(rng, dtype, 16, 3)
    q, k, v, dout = (tensor(rng, dtype, n, 3, 32) for _ in range(4))
    out, lse = layers.attention(q, k, v, plan, table=table, buckets=b)
    want = layers.attention_backward(dout, q, k, v, out, lse, plan, table=table, buckets=b)
    for split in ((lambda t: [t[:, 3 * i:3 * i + 3] for i in range(4)]), (lambda t: [t.view(n + 2, 3, 4, 32)[:, :, i] for i in range(4)])):
        x, g = (torch.full((n + 2, 12, 32), 5.0, dtype=q.dtype, device="cuda") for _ in range(2))
        for to, t in zip(split(x), (q, k, v, dout)):
            to[:n].copy_(t)
        qs, ks, vs, ds = split(x)
        dq, dk, dv, spare = split(g)
        o, l = layers.attention(qs, ks, vs, plan, table=table, buckets=b)
        dt = layers.attention_backward(ds, qs, ks, vs, o, l, plan, table=table, buckets=b, dq=dq, dk=dk, dv=dv)[3]
        for a, c in zip((o, l, dq[:n], dk[:n], dv[:n], dt), (out, lse) + want):
            assert torch.equal(a, c)
        assert (spare == 5.0).all() and (g[n:] == 5.0).all()
