"""Layer operators without a GPU: the attention plan covers what it has to, tables are what they say, bad calls are refused."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from deepptmpred_amd import _native, layers  # noqa: E402
from oracle import layers_ref as R  # noqa: E402

Q_ITEM, K_ITEM, JOIN = 8, 12, 4


def see(q_lens, k_lens, window, sinks, pos):
    """Visible pairs of packed rows and packed keys."""
    m = np.zeros((sum(q_lens), sum(k_lens)), bool)
    q0 = k0 = 0
    for a, b in zip(q_lens, k_lens):
        p, j = pos[q0:q0 + a][:, None], np.arange(b)[None]
        v = np.ones((a, b), bool)
        if window[1] >= 0:
            v &= j <= p + window[1]
        if window[0] >= 0:
            v &= (j >= p - window[0]) | (j < sinks)
        m[q0:q0 + a, k0:k0 + b] = v
        q0, k0 = q0 + a, k0 + b
    return m


BATCHES = [([], []), ([0], [0]), ([1], [1]), ([5, 0, 200], [5, 0, 200]), ([1, 1, 1], [700, 0, 3000]), ([40, 3], [10, 500]),
           ([129, 64, 1], [129, 64, 1]), ([53], [2000])]


@pytest.mark.parametrize("q_lens,k_lens", BATCHES)
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((-1, 0), 0), ((20, 7), 3), ((0, 0), 40), ((5, -1), 2), ((300, 0), 130)])
@pytest.mark.parametrize("heads", [1, 64, (24, 4)])
@pytest.mark.parametrize("given", [False, True])
def test_plan_covers_every_visible_pair_once(q_lens, k_lens, window, sinks, heads, given):
    rng = np.random.default_rng(sum(k_lens) + sinks)
    pos = np.concatenate([rng.integers(-3, b + 3, a) for a, b in zip(q_lens, k_lens)] or [np.zeros(0)]).astype(np.int32) if given else None
    heads, kv_heads = heads if isinstance(heads, tuple) else (heads, heads)
    plan = layers.AttentionPlan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, head_dim=32, window=window, sinks=sinks, q_positions=pos, device=None)
    w = plan.words
    assert heads // kv_heads % w[30] == 0 and w[30] * min(32, max(q_lens, default=0)) <= 32 * (w[30] > 1) + 32 * (w[30] == 1)
    p = pos if given else R.default_positions(q_lens, k_lens)
    m = see(q_lens, k_lens, window, sinks, p)
    starts = {}
    q0 = k0 = 0
    for a, b in zip(q_lens, k_lens):
        for i in range(a):
            starts[q0 + i] = (k0, b)
        q0, k0 = q0 + a, k0 + b
    # forward and dq: every row's visible keys lie in the ranges of its items, each once; parts are joined
    for at, n, tile in ((w[13], w[12], (128, 64, 32 // w[30])[w[11]]), (w[18], w[17], 32 * w[19])):
        count = np.zeros(m.shape, np.int64)
        slots = []
        for it in w[at:at + Q_ITEM * n].reshape(-1, Q_ITEM):
            first, nq, ks, pos0, kb, ke, sink_end, slot = (int(v) for v in it)
            assert 1 <= nq <= tile
            for r in range(first, first + nq):
                base, length = starts[r]
                assert ks == base and 0 <= kb <= ke <= length and 0 <= sink_end <= kb
                if not given:
                    assert p[r] == pos0 + r - first
                count[r, ks + kb:ks + ke] += 1
                count[r, ks:ks + sink_end] += 1
            if slot >= 0:
                slots.append(slot)
        assert count.max(initial=0) <= 1 and not (m & (count == 0)).any()
        rows = np.zeros(len(m), np.int64)
        for it in w[at:at + Q_ITEM * n].reshape(-1, Q_ITEM):
            if it[7] < 0:
                rows[it[0]:it[0] + it[1]] += 1
        if at == w[13]:
            joined = []
            for first, nq, slot0, k in w[w[16]:w[16] + JOIN * w[15]].reshape(-1, JOIN):
                rows[first:first + nq] += 1
                joined += list(range(slot0, slot0 + k))
            assert sorted(slots) == sorted(joined) == list(range(w[14]))
        assert (rows == 1).all()
    # dk, dv: the other way round
    count = np.zeros(m.shape, np.int64)
    keys = np.zeros(m.shape[1], np.int64)
    slots = []
    for it in w[w[21]:w[21] + K_ITEM * w[20]].reshape(-1, K_ITEM):
        first, nk, j0, q0, qb, qe, pos0, slot, tile0, nseq = (int(v) for v in it[:10])
        assert 1 <= nk <= 32 * w[22] and qb % 32 == 0 and 0 <= qb <= qe <= nseq
        count[q0 + qb:q0 + qe, first:first + nk] += 1
        if slot < 0:
            keys[first:first + nk] += 1
        else:
            slots.append(slot)
        if given:
            for i in range(qb, qe, 32):
                lo, hi = w[w[29] + 2 * (tile0 + i // 32)], w[w[29] + 2 * (tile0 + i // 32) + 1]
                assert lo == p[q0 + i:q0 + min(i + 32, nseq)].min() and hi == p[q0 + i:q0 + min(i + 32, nseq)].max()
    joined = []
    for first, nk, slot0, k in w[w[25]:w[25] + JOIN * w[24]].reshape(-1, JOIN):
        keys[first:first + nk] += 1
        joined += list(range(slot0, slot0 + k))
    assert sorted(slots) == sorted(joined) == list(range(w[23]))
    assert (keys == 1).all() and count.max(initial=0) <= 1 and not (m & (count == 0)).any()


def test_long_sequences_split_evenly():
    """One long sequence under a window with first tokens: no tile of keys keeps a range of rows far longer than the others'."""
    plan = layers.AttentionPlan([16001], heads=8, head_dim=64, window=(512, 512), sinks=1, device=None)
    w = plan.words
    rows = [int(it[5] - it[4]) for it in w[w[21]:w[21] + K_ITEM * w[20]].reshape(-1, K_ITEM)]
    assert max(rows) <= 4 * np.median(rows)


def test_relative_buckets():
    m = layers.relative_buckets(32, 128, device=None)
    assert m.dtype == np.int32 and m.shape == (257,)
    at = lambda d: int(m[128 + d])  # noqa: E731
    assert [at(-d) for d in range(9)] == list(range(9)) and [at(d) for d in range(1, 9)] == list(range(17, 25))
    assert at(0) == 0 and at(-128) == 15 and at(128) == 31
    # 8 (128 / 8)^(k / 8) = 8 2^(k / 2): borders at 11.3, 16, 22.6, 32, 45.3, 64, 90.5
    assert [at(-d) for d in (11, 12, 15, 16, 22, 23, 31, 32, 45, 46, 63, 64, 90, 91)] == [8, 9, 9, 10, 10, 11, 11, 12, 12, 13, 13, 14, 14, 15]
    b = layers.relative_buckets(8, 20, False, device=None)
    assert (b[20:] == 0).all() and b[0] == 7 and (np.diff(b) <= 0).all() and set(b) == set(range(8))
    for bad in ((3, 9, True), (2, 9, True), (66, 128, True), (32, 8, True), (32, 1025, True), (1, 9, False)):
        with pytest.raises(ValueError):
            layers.relative_buckets(*bad, device=None)


def test_rotary_table():
    cos, sin = layers.rotary_table(5000, 64, device="cpu")
    assert cos.shape == sin.shape == (5000, 32) and cos.dtype == torch.float32
    a = 4999 * 10000.0 ** (-2 * 7 / 64)
    assert abs(float(cos[4999, 7]) - np.cos(a)) < 1e-7 and abs(float(sin[4999, 7]) - np.sin(a)) < 1e-7
    with pytest.raises(ValueError):
        layers.rotary_table(10, 7, device="cpu")


def test_plan_refusals():
    ok = dict(heads=4, head_dim=64, device=None)
    for bad, more in (([5], dict(head_dim=48)), ([5], dict(heads=4, kv_heads=3)), ([5], dict(heads=0)), ([5], dict(sinks=-1)),
                      ([-1], {}), ([2 ** 29], {}), ([2 ** 28] * 8 + [7] * 2, {}), ([5], dict(q_positions=[0, 1, 2])),
                      ([2], dict(q_positions=[0, 2 ** 29])), ([5], dict(k_lens=[5, 5])), ([[5]], {}), ([5.5], {}),
                      ([2 ** 40], {}), ([5], dict(heads=5000))):
        with pytest.raises(ValueError):
            layers.AttentionPlan(bad, **{**ok, **more})
    assert layers.AttentionPlan([], **ok).q_rows == 0


def rows_of(n, heads, dim, at=1 << 20, size=2):
    return _native.Rows(at, n, heads * dim, dim)


def test_c_calls_are_refused_before_anything_runs():
    """Bad sizes, strides, addresses and plans come back as DPTM_EINVAL: none of these addresses is ever touched."""
    lib = _native.load_library()
    plan = layers.AttentionPlan([10], heads=2, head_dim=64, device=None)
    P = plan.words.ctypes.data
    good = rows_of(10, 2, 64)

    def forward(plan_host=P, dtype=1, q=good, k=good, v=good, out=good, lse=1 << 20, scale=0.1, bias=(0, 0, 0, 0), ws=None, ws_bytes=0):
        x = _native.AttentionArgs(plan=plan_host, plan_dev=P, q=q, k=k, v=v, out=out, lse=lse, table=bias[0], buckets=bias[1],
                                  workspace=ws, workspace_bytes=ws_bytes, dtype=dtype, n_buckets=bias[2], max_distance=bias[3], scale=scale)
        return lib.dptm_attention_forward(C.addressof(x))

    def says(rc, text):
        assert rc == _native.DPTM_EINVAL and text in lib.dptm_layer_last_error().decode(), lib.dptm_layer_last_error()

    need = lib.dptm_attention_workspace(P, 0, 0, 0)
    ws = dict(ws=1 << 20, ws_bytes=need)
    says(forward(plan_host=None, **ws), "NULL plan")
    other = plan.words.copy()
    other[12] += 1
    says(forward(plan_host=other.ctypes.data, **ws), "not a plan")
    says(forward(dtype=3, **ws), "dtype")
    says(forward(scale=0.0, **ws), "scale")
    says(forward(scale=-1.0, **ws), "scale")
    says(forward(scale=float("nan"), **ws), "scale")
    says(forward(q=_native.Rows(None, 10, 128, 64), **ws), "NULL buffer")
    says(forward(k=rows_of(9, 2, 64), **ws), "k has 9 rows")
    says(forward(v=rows_of(10, 2, 64, at=(1 << 20) + 8), **ws), "16 bytes")
    says(forward(q=_native.Rows(1 << 20, 10, 132, 64), **ws), "16 bytes")
    says(forward(q=_native.Rows(1 << 20, 10, -128, 64), **ws), "negative")
    says(forward(out=_native.Rows(1 << 20, 10, 64, 64), **ws), "overlap")
    says(forward(out=_native.Rows(1 << 20, 10, 128, 0), **ws), "overlap")
    says(forward(lse=None, **ws), "lse")
    if need:
        says(forward(), "workspace")
        says(forward(ws=(1 << 20) + 16, ws_bytes=need), "256-byte")
    at = 1 << 20
    for n, far in ((0, 5), (65, 5), (8, -1), (8, 1025)):
        says(forward(bias=(at, at, n, far), **ws), "supported")
    says(forward(bias=(0, at, 8, 9), **ws), "together")
    says(forward(bias=(at, 0, 8, 9), **ws), "together")
    says(forward(bias=(at + 1, at, 8, 9), **ws), "aligned")
    says(forward(bias=(at, at + 2, 8, 9), **ws), "aligned")

    def backward(plan_host=P, dq=good, dk=good, bias=(0, 0, 0, 0), dtable=None, ws=1 << 20, ws_bytes=1 << 30, lse=1 << 20):
        x = _native.AttentionArgs(plan=plan_host, plan_dev=P, q=good, k=good, v=good, out=good, lse=lse, table=bias[0], buckets=bias[1],
                                  workspace=ws, workspace_bytes=ws_bytes, dout=good, dq=dq, dk=dk, dv=good, dtable=dtable, dtype=1,
                                  n_buckets=bias[2], max_distance=bias[3], scale=0.1)
        return lib.dptm_attention_backward(C.addressof(x))

    says(backward(ws_bytes=16), "workspace")
    says(backward(dq=_native.Rows(1 << 20, 10, 128, 0)), "overlap")
    says(backward(dk=rows_of(3, 2, 64)), "dk has 3 rows")
    says(backward(bias=(at, at, 8, 9)), "gradient")
    says(backward(lse=None), "lse")
    fwd_only = layers.AttentionPlan([10], heads=2, head_dim=64, training=False, device=None)
    says(backward(plan_host=fwd_only.words.ctypes.data), "without training")
    says(lib.dptm_attention_forward(None), "NULL arguments")
    says(lib.dptm_attention_backward(None), "NULL arguments")
    says(lib.dptm_attention_workspace(None, 0, 0, 0), "NULL plan")
    says(lib.dptm_attention_workspace(P, 65, 0, 0), "supported")
    says(lib.dptm_attention_workspace(P, 8, 1025, 0), "supported")
    assert lib.dptm_attention_plan(None, None, None, None, 0, None, 0) == _native.DPTM_EINVAL


def test_argument_blocks_match_the_header():
    """The packed form of the argument blocks has the layout of the structures, which is the header's."""
    assert layers._NORM_ROPE.size == C.sizeof(_native.NormRopeArgs)
    a = _native.AttentionArgs
    assert layers._ATTENTION.size == a.scale.offset + 4 and C.sizeof(a) == (layers._ATTENTION.size + 7) // 8 * 8
    words = list(range(1, 1 + 2 + 16 + 6 + 16 + 1)) + [1, 2, 3, 4, 0.5]
    x = a.from_buffer_copy(layers._ATTENTION.pack(*words) + b"\0" * 8)
    assert (x.plan, x.plan_dev, x.q.data, x.out.head_stride, x.lse, x.stream, x.dout.data, x.dv.head_stride, x.dtable) == \
        (1, 2, 3, 18, 19, 24, 25, 40, 41)
    assert (x.dtype, x.device, x.n_buckets, x.max_distance, x.scale) == (1, 2, 3, 4, 0.5)
    y = _native.NormRopeArgs.from_buffer_copy(layers._NORM_ROPE.pack(*range(1, 51), 0.25))
    assert (y.q.data, y.k_out.head_stride, y.q_gain, y.stream, y.dq_out.data, y.dk.head_stride, y.dq_gain, y.rows, y.dtype, y.eps) == \
        (1, 16, 17, 22, 23, 38, 39, 43, 44, 0.25) and y.interleaved == 50


def test_c_norm_calls_are_refused_before_anything_runs():
    lib = _native.load_library()
    good = rows_of(10, 2, 64)
    tab = 1 << 20

    def args(**more):
        return _native.NormRopeArgs(**{**dict(q=good, k=good, q_out=good, k_out=good, q_gain=tab, k_gain=tab, cosv=tab, sinv=tab, dq_out=good,
                                              dk_out=good, dq=good, dk=good, dtype=1, head_dim=64, heads=2, kv_heads=2, rows=10,
                                              n_positions=10, eps=1e-6), **more})

    def says(rc, text):
        assert rc == _native.DPTM_EINVAL and text in lib.dptm_layer_last_error().decode(), (text, lib.dptm_layer_last_error())

    for bad, text in ((dict(dtype=7), "dtype"), (dict(head_dim=24), "head_dim"), (dict(heads=-1), "heads"),
                      (dict(heads=0, kv_heads=0), "heads"), (dict(rows=-1), "row"), (dict(eps=-1.0), "eps"),
                      (dict(eps=float("nan")), "eps"), (dict(n_positions=-1), "positions"), (dict(cosv=None), "cos"),
                      (dict(cosv=tab + 4), "16-byte"), (dict(q_gain=tab + 4), "aligned"), (dict(positions=tab + 2), "aligned"),
                      (dict(q=rows_of(9, 2, 64)), "rows"), (dict(q_out=_native.Rows(tab, 10, 128, 0)), "overlap"),
                      (dict(k=_native.Rows(None, 10, 128, 64)), "NULL"), (dict(rows=2 ** 31), "row")):
        x = args(**bad)
        says(lib.dptm_qk_norm_rope_forward(C.addressof(x)), text)
    for bad, text in ((dict(), "gradient"), (dict(dq_gain=tab, dk_gain=tab), "workspace"),
                      (dict(dq=_native.Rows(tab, 10, 128, 0)), "overlap")):
        x = args(**bad)
        says(lib.dptm_qk_norm_rope_backward(C.addressof(x)), text)
    says(lib.dptm_qk_norm_rope_forward(None), "NULL arguments")
    says(lib.dptm_qk_norm_rope_backward(None), "NULL arguments")
    says(lib.dptm_qk_norm_rope_workspace(None), "sizes")


def test_python_refusals():
    plan = layers.AttentionPlan([4], heads=2, head_dim=16, device=None)
    t = torch.zeros(4, 2, 16)
    for bad in ((t, t, t), (t.double(), t, t), (np.zeros((4, 2, 16), np.float32), t, t)):
        with pytest.raises(ValueError):
            layers.attention(*bad, plan)
    with pytest.raises(ValueError):
        layers.qk_norm_rope(t, t, torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError):
        layers.qk_norm_rope(t, t[:3], torch.zeros(4, 8), torch.zeros(4, 8))


@pytest.mark.parametrize("window,sinks,buckets", [((-1, -1), 0, False), ((3, 1), 2, True), ((2, 0), 0, True)])
def test_the_restated_gradients_are_the_differences_of_the_forward_pass(window, sinks, buckets):
    rng = np.random.default_rng(4)
    q_lens, k_lens = [5, 3, 1], [7, 3, 0]
    x = {"q": rng.normal(size=(9, 4, 6)), "k": rng.normal(size=(10, 2, 6)), "v": rng.normal(size=(10, 2, 6)), "table": rng.normal(size=(4, 4))}
    of = np.array([0, 1, 2, 3, 3]) if buckets else None
    w = rng.normal(size=(9, 4, 6))

    def loss(y, dout=None):
        return R.attention(y["q"], y["k"], y["v"], q_lens, k_lens, window, sinks, None, None, y["table"] if buckets else None, of, dout)

    r = loss(x, w)
    for n, g in (("q", "dq"), ("k", "dk"), ("v", "dv")) + ((("table", "dtable"),) if buckets else ()):
        d = rng.normal(size=x[n].shape)
        up, down = {**x, n: x[n] + 1e-6 * d}, {**x, n: x[n] - 1e-6 * d}
        slope = ((loss(up)["out"][0] - loss(down)["out"][0]) * w).sum() / 2e-6
        assert abs(slope - (r[g][0] * d).sum()) < 1e-6, n
    cos, sin = np.cos(rng.normal(size=(9, 3))), np.sin(rng.normal(size=(9, 3)))
    gain = rng.normal(size=6)
    for inter in (False, True):
        for gn in (gain, None):
            f = lambda y, dy=None, gg=gn: R.qk_norm_rope(y, gg, cos, sin, np.arange(9), 1e-3, inter, dy)  # noqa: E731
            r = f(x["q"], w)
            d = rng.normal(size=x["q"].shape)
            slope = ((f(x["q"] + 1e-6 * d)["y"][0] - f(x["q"] - 1e-6 * d)["y"][0]) * w).sum() / 2e-6
            assert abs(slope - (r["dx"][0] * d).sum()) < 1e-6
            if gn is not None:
                d = rng.normal(size=6)
                slope = ((f(x["q"], None, gn + 1e-6 * d)["y"][0] - f(x["q"], None, gn - 1e-6 * d)["y"][0]) * w).sum() / 2e-6
                assert abs(slope - (r["dgain"][0] * d).sum()) < 1e-6


def test_results_that_share_memory_with_others_are_refused():
    """What a call writes lies apart from what it reads and from what else it writes; columns of one packed tensor do."""
    lib = _native.load_library()
    plan = layers.AttentionPlan([10], heads=2, head_dim=64, device=None)
    P, n = plan.words.ctypes.data, 1 << 22

    def packed(part, row=6 * 64, head=64):     # two heads of a tensor [10][q k v][64], bfloat16
        return _native.Rows((1 << 24) + part * 2 * 64 * 2, 10, row, head)

    def forward(out, q=packed(0), k=packed(1), v=packed(2)):
        x = _native.AttentionArgs(plan=P, plan_dev=P, q=q, k=k, v=v, out=out, lse=n, dtype=1, scale=0.1, device=4096, workspace=n, workspace_bytes=n)
        return lib.dptm_attention_forward(C.addressof(x))

    def says(rc, text):
        assert rc == _native.DPTM_EINVAL and text in lib.dptm_layer_last_error().decode(), (text, lib.dptm_layer_last_error())

    apart = "no such device"                   # the last check before anything runs
    says(forward(rows_of(10, 2, 64, at=1 << 20)), apart)
    for part, name in enumerate("qkv"):
        says(forward(packed(part)), f"out shares memory with {name}")
    says(forward(packed(1), k=packed(2)), apart)
    says(forward(rows_of(10, 2, 64, at=(1 << 24) + 9 * 6 * 128)), "shares memory")                     # inside the last row
    says(forward(rows_of(10, 2, 64, at=(1 << 24) + (9 * 6 + 6) * 128)), apart)                         # right behind it
    says(forward(_native.Rows((1 << 24) + 128, 10, 128, 64), *(rows_of(10, 2, 64, at=(1 << 24)),) * 3), "out shares memory with q")
    # [row][head][q k v][64]
    by_head = [_native.Rows((1 << 24) + part * 128, 10, 6 * 64, 3 * 64) for part in range(3)]
    says(forward(by_head[1], by_head[0], by_head[2], by_head[2]), apart)
    says(forward(by_head[1], by_head[0], by_head[1], by_head[2]), "out shares memory with k")
    says(forward(_native.Rows((1 << 24) + 64, 10, 6 * 64, 3 * 64), *by_head), "shares memory")

    def backward(dq=packed(0), dk=packed(1), dv=packed(2)):
        some = rows_of(10, 2, 64, at=1 << 20)
        x = _native.AttentionArgs(plan=P, plan_dev=P, q=some, k=some, v=some, out=some, lse=n, workspace=1 << 30, workspace_bytes=1 << 30, dout=some,
                                  dq=dq, dk=dk, dv=dv, dtype=1, scale=0.1, device=4096)
        return lib.dptm_attention_backward(C.addressof(x))

    says(backward(), apart)
    says(backward(dk=packed(0)), "dq shares memory with dk")
    says(backward(dv=packed(1)), "dk shares memory with dv")
    says(backward(dv=rows_of(10, 2, 64, at=1 << 20)), "dv shares memory with q")

    def norm(back=False, **more):
        x = _native.NormRopeArgs(**{**dict(q=packed(0), k=packed(1), q_out=packed(0), k_out=packed(1), cosv=n, sinv=n, dq_out=packed(2, 8 * 64),
                                           dk_out=packed(3, 8 * 64), dq=packed(2, 8 * 64), dk=packed(3, 8 * 64), dtype=1, head_dim=64, heads=2,
                                           kv_heads=2, rows=10, n_positions=10, eps=1e-6, device=4096), **more})
        if back:
            x.q, x.k = rows_of(10, 2, 64, at=1 << 20), rows_of(10, 2, 64, at=1 << 21)
        return (lib.dptm_qk_norm_rope_backward if back else lib.dptm_qk_norm_rope_forward)(C.addressof(x))

    says(norm(), apart)                        # in place
    says(norm(q_out=packed(2)), apart)
    says(norm(q_out=packed(1), k_out=packed(0)), "shares memory")
    says(norm(k_out=packed(0)), "shares memory")
    says(norm(q_out=packed(0, 7 * 64)), "q_out shares memory with")
    says(norm(back=True), apart)
    says(norm(back=True, dq=packed(3, 8 * 64)), "shares memory")


def test_sizes_that_no_launch_or_offset_holds_are_refused():
    lib = _native.load_library()
    plan = layers.AttentionPlan([10], heads=2, head_dim=64, device=None)
    P, n = plan.words.ctypes.data, 1 << 22

    def forward(scale=0.1, **more):
        x = _native.AttentionArgs(**{**dict(plan=P, plan_dev=P, q=rows_of(10, 2, 64), k=rows_of(10, 2, 64), v=rows_of(10, 2, 64), lse=n, dtype=0,
                                            out=rows_of(10, 2, 64, at=1 << 24), device=4096, workspace=n, workspace_bytes=n), **more}, scale=scale)
        return lib.dptm_attention_forward(C.addressof(x))

    def says(rc, text):
        assert rc == _native.DPTM_EINVAL and text in lib.dptm_layer_last_error().decode(), (text, lib.dptm_layer_last_error())

    for row in (1 << 23, 1 << 40, 1 << 62, (1 << 62) + 128):                # 32 MiB and more, also where the bytes wrap
        says(forward(q=_native.Rows(1 << 20, 10, row, 64)), "32 MiB")
    says(forward(q=_native.Rows(1 << 20, 10, (1 << 23) - 4, 64)), "no such device")
    says(forward(v=_native.Rows(1 << 20, 10, 128, 1 << 62)), "32 MiB")
    for scale in (1e-20, 1e-39, 1e20, float("inf")):
        says(forward(scale=scale), "scale")
    # threads of a launch are counted in 32 bits: 4,096 heads, tiles of 128 rows
    with pytest.raises(ValueError, match="one launch"):
        layers.AttentionPlan([128] * 4096, heads=4096, head_dim=16, training=False, device=None)
    layers.AttentionPlan([128] * 4095, heads=4096, head_dim=16, training=False, device=None)
    x = _native.NormRopeArgs(q=rows_of(2 ** 24, 256, 16), k=rows_of(2 ** 24, 1, 16), dtype=1, head_dim=16, heads=256, kv_heads=1, rows=2 ** 24,
                             cosv=n, sinv=n, eps=1e-6, device=4096)
    says(lib.dptm_qk_norm_rope_forward(C.addressof(x)), "one launch")


def test_a_bias_that_is_no_tensor_is_refused():
    plan = layers.AttentionPlan([5], heads=2, head_dim=16, device=None)
    with pytest.raises(ValueError, match="torch tensors"):
        layers._bias("attention", plan, np.zeros((8, 2), np.float32), layers.relative_buckets(8, 20, device=None), torch.float32, 0)


def test_keys_out_of_reach_of_a_window_without_limit_are_refused():
    """A side without limit reaches 2^29 positions: a batch whose keys lie further ahead would lose them without a word."""
    ok = dict(heads=1, head_dim=64, device=None)
    far = 2 ** 29
    for window in ((-1, -1), (7, -1), (-1, 2 ** 31 - 1)):
        with pytest.raises(ValueError, match="2\\^29"):
            layers.AttentionPlan([1], [100], q_positions=[-far + 1], window=window, **ok)
        with pytest.raises(ValueError, match="2\\^29"):
            layers.AttentionPlan([3, 2], [7, 100], q_positions=[0, 1, 2, 50, -far + 98], window=window, **ok)
    # the last that is in reach sees all of its keys, and so do rows that are limited or far behind
    for position, window, keys in ((-far + 99, (-1, -1), 100), (far - 1, (-1, -1), 100), (-far + 1, (-1, 5), 0), (far - 1, (-1, 0), 100)):
        w = layers.AttentionPlan([1], [100], q_positions=[position], window=window, **ok).words
        assert [int(x) for x in w[w[13] + 4:w[13] + 6]] == [0, keys] and w[12] == 1
    assert layers.AttentionPlan([0, 1], [far - 1, 4], window=(-1, -1), **ok).k_rows == far + 3


def test_shared_memory_is_found_byte_by_byte():
    """Random layouts -- head-major, packed, repeated, larger or smaller than each other -- against the sets of their bytes."""
    lib = _native.load_library()
    rng = np.random.default_rng(7)
    base, seen = 1 << 24, {True: 0, False: 0}

    def layout(rows, heads):
        kind = rng.integers(0, 5)
        gap = lambda most: 8 * int(rng.integers(0, most))                       # elements of two bytes, steps of 16 bytes  # noqa: E731
        if kind < 2:
            head = 16 + gap(8)
            return heads * head + gap(8), head
        if kind < 4:
            row = 16 + gap(8)
            return row, rows * row + gap(8)
        return [(0, 16), (16, 0), (8, 24), (0, 0)][rng.integers(0, 4)]          # for what is read alone

    def touched(at, rows, heads, row, head):
        return {at + 2 * (i * row + j * head) + b for i in range(rows) for j in range(heads) for b in range(0, 32, 16)}

    for _ in range(4000):
        nq, nk, heads, kv = int(rng.integers(1, 5)), int(rng.integers(1, 6)), 2, int(rng.integers(1, 3))
        plan = layers.AttentionPlan([nq], [nk], heads=heads, kv_heads=kv, head_dim=16, device=None)
        P = plan.words.ctypes.data
        (orow, ohead), (krow, khead) = layout(nq, heads), layout(nk, kv)
        out, k = base, base + 16 * int(rng.integers(-30, 30))
        far = _native.Rows(1 << 26, 8, 64, 16)
        x = _native.AttentionArgs(plan=P, plan_dev=P, q=far, k=_native.Rows(k, nk, krow, khead), v=far, out=_native.Rows(out, nq, orow, ohead), lse=1 << 27,
                                  dtype=1, scale=0.1, device=4096, workspace=1 << 28, workspace_bytes=1 << 20)
        rc, said = lib.dptm_attention_forward(C.addressof(x)), lib.dptm_layer_last_error().decode()
        assert rc == _native.DPTM_EINVAL
        if "overlap" in said:
            continue                                                            # no layout for what is written
        shared = bool(touched(out, nq, heads, orow, ohead) & touched(k, nk, kv, krow, khead))
        seen[shared] += 1
        assert ("out shares memory with k" in said) == shared and ("no such device" in said) != shared, (said, nq, nk, kv, orow, ohead, krow, khead, k - out)
    assert min(seen.values()) > 300


def test_every_buffer_that_a_call_writes_lies_apart():
    """Head-major tensors, lse, tables, gradients of tables and gains, and the workspace."""
    lib = _native.load_library()
    plan = layers.AttentionPlan([10, 300], heads=2, head_dim=64, device=None)
    P, n, u = plan.words.ctypes.data, 310, 1 << 22
    at = {name: (i + 4) * u for i, name in enumerate("q k v out dout dq dk dv lse table buckets dtable ws".split())}

    def said(call, **moved):
        a = {**at, **moved}
        r = {x: _native.Rows(a[x], n, 64, n * 64) for x in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")}      # [heads][rows][64]
        x = _native.AttentionArgs(plan=P, plan_dev=P, lse=a["lse"], table=a["table"], buckets=a["buckets"], dtable=a["dtable"], workspace=a["ws"], workspace_bytes=u,
                                  dtype=1, scale=0.1, device=4096, n_buckets=8, max_distance=20, **r)
        assert call(C.addressof(x)) == _native.DPTM_EINVAL
        return lib.dptm_layer_last_error().decode()

    fwd, bwd = lib.dptm_attention_forward, lib.dptm_attention_backward
    need = [lib.dptm_attention_workspace(P, 8, 20, b) for b in (0, 1)]
    apart = "no such device"                   # at the end of what is said, the last check before anything runs
    assert said(fwd).endswith(apart) and said(bwd).endswith(apart) and need[1] > 1000
    head = n * 64 * 2
    assert "out shares memory with q" in said(fwd, out=at["q"] + head)                  # one head on
    assert "out shares memory with q" in said(fwd, out=at["q"] + 128)
    assert said(fwd, out=at["q"] + 2 * head).endswith(apart)
    assert "lse" in said(fwd, lse=at["q"] + 256) and "lse" in said(fwd, lse=at["out"] + 256)
    assert "out shares memory with table" in said(fwd, table=at["out"] + 64) and "buckets" in said(fwd, buckets=at["out"] + 2 * head - 4)
    assert said(fwd, buckets=at["out"] + 2 * head).endswith(apart)
    assert "out shares memory with plan" in said(fwd, out=(P + 15) // 16 * 16)
    for other in ("q", "k", "v", "out", "dout", "lse", "table", "buckets", "dtable", "ws", "dk"):
        assert f"dq shares memory with {'workspace' if other == 'ws' else other}" in said(bwd, dq=at[other])
        if other not in ("dtable", "dk"):
            assert "dtable shares memory with" in said(bwd, dtable=at[other])
        if other not in ("ws", "dk", "dtable"):
            assert f"workspace shares memory with {other}" in said(bwd, ws=at[other])
    assert "workspace shares memory with q" in said(bwd, ws=(at["q"] - need[1]) // 256 * 256 + 256)
    assert said(bwd, ws=(at["q"] - need[1]) // 256 * 256).endswith(apart)

    def norm(back, **moved):
        names = "q k q_out k_out dq_out dk_out dq dk".split()
        a = {x: (i + 4) * u for i, x in enumerate(names + "q_gain k_gain cosv sinv positions dq_gain dk_gain workspace".split())}
        a.update(moved)
        x = _native.NormRopeArgs(**{**a, **{x: _native.Rows(a[x], 40, 64, 40 * 64) for x in names}}, workspace_bytes=u, rows=40, dtype=1, device=4096, head_dim=64,
                                 heads=2, kv_heads=2, n_positions=40, eps=1e-6)
        assert (lib.dptm_qk_norm_rope_backward if back else lib.dptm_qk_norm_rope_forward)(C.addressof(x)) == _native.DPTM_EINVAL
        return lib.dptm_layer_last_error().decode()

    assert norm(False).endswith(apart) and norm(True).endswith(apart)
    assert norm(False, q_out=4 * u).endswith(apart) and norm(True, dq=4 * u).endswith(apart) and norm(True, dq=8 * u).endswith(apart)
    assert "q_out shares memory with q" in norm(False, q_out=4 * u + 40 * 128)
    for x in ("q_gain", "k_gain", "cosv", "sinv", "positions"):
        assert "q_out shares memory" in norm(False, **{x: 6 * u + 128}) and "dk shares memory" in norm(True, **{x: 11 * u + 2 * 40 * 128 - 16})
    for x in ("dq_gain", "dk_gain", "workspace"):
        for y in range(4, 17):
            if y not in (6, 7):                                                         # q_out, k_out: the forward call's
                assert "shares memory with" in norm(True, **{x: y * u}), (x, y)
    assert "dq_gain shares memory with dk_gain" in norm(True, dq_gain=18 * u) and "aligned" in norm(True, dq_gain=17 * u + 2)
    # the same memory in another order is not in place
    x = _native.NormRopeArgs(q=_native.Rows(u, 40, 64, 40 * 64), q_out=_native.Rows(u, 40, 128, 64), cosv=2 * u, sinv=3 * u, rows=40, dtype=1, device=4096,
                             head_dim=64, heads=2, kv_heads=0, n_positions=40, eps=1e-6)
    assert lib.dptm_qk_norm_rope_forward(C.addressof(x)) == _native.DPTM_EINVAL and b"q_out shares memory with q" in lib.dptm_layer_last_error()


def test_numbers_that_the_argument_blocks_do_not_hold():
    """Sizes are refused, not cut to 32 bits; more first tokens, or a wider window, than any sequence is long are all of them."""
    ok = dict(heads=4, head_dim=64, device=None)
    for bad in (dict(heads=2 ** 32 + 4), dict(kv_heads=2 ** 32 + 4), dict(head_dim=2 ** 32 + 64), dict(heads=2.5), dict(sinks=1.5), dict(sinks=-2 ** 40),
                dict(window=(1.5, 0)), dict(window=(float("inf"), 0)), dict(window=3), dict(window=(None, 0)), dict(heads=None), dict(device="cpu")):
        with pytest.raises(ValueError, match="AttentionPlan"):
            layers.AttentionPlan([5], **{**ok, **bad})
    every = layers.AttentionPlan([500], window=(3, 0), sinks=500, **ok).words
    for many in (2 ** 32 + 1, 2 ** 31, 10 ** 6):
        w = layers.AttentionPlan([500], window=(3, 0), sinks=many, **ok).words
        assert np.array_equal(w[w[13]:w[18]], every[every[13]:every[18]]) and w[7] >= 500
    w = layers.AttentionPlan([5], window=(2 ** 40, -2 ** 40), **ok).words
    assert list(w[5:7]) == [2 ** 29] * 2
    assert layers.AttentionPlan([5], **{**ok, "heads": np.int64(4), "window": (np.int32(2), 2.0)}).words[5] == 2
    for bad in ((32.5, 128), (32, 128.5), (2 ** 40, 128), (32, "x")):
        with pytest.raises(ValueError):
            layers.relative_buckets(*bad, device=None)
    for bad in ((5.5, 64, 1e4), (5, 64.5, 1e4), (5, 64, -3.0), (5, 64, 0.0), (5, 64, float("nan"))):
        with pytest.raises(ValueError):
            layers.rotary_table(*bad, device="cpu")
    for bad in (1e39, -1e39, float("inf"), float("nan"), 10 ** 400):
        with pytest.raises(ValueError, match="eps"):
            layers._f32(bad, "qk_norm_rope", "eps")
    assert layers._f32(np.float32(0.125), "attention", "scale") == 0.125


def test_c_sizes_and_addresses_at_their_limits():
    """Sizes that no call takes have no workspace, and a plan at an odd address is no plan."""
    lib = _native.load_library()

    def workspace(**more):
        x = _native.NormRopeArgs(**{**dict(rows=100, heads=4, kv_heads=4, head_dim=64), **more})
        return lib.dptm_qk_norm_rope_workspace(C.addressof(x))

    assert workspace() > 0 and workspace(rows=0) > 0 and workspace(rows=2 ** 31 - 1) == 1536 * 64 * 8
    for bad in (dict(rows=2 ** 31), dict(rows=2 ** 62), dict(heads=2 ** 31 - 1), dict(kv_heads=4097), dict(head_dim=48)):
        assert workspace(**bad) == _native.DPTM_EINVAL and b"sizes" in lib.dptm_layer_last_error()
    plan = layers.AttentionPlan([10], heads=2, head_dim=64, device=None)
    P = plan.words.ctypes.data
    good = rows_of(10, 2, 64)
    x = _native.AttentionArgs(plan=P, plan_dev=P + 2, q=good, k=good, v=good, out=rows_of(10, 2, 64, at=1 << 24), lse=1 << 25, dtype=1, scale=0.1, device=4096,
                              workspace=1 << 26, workspace_bytes=1 << 20)
    assert lib.dptm_attention_forward(C.addressof(x)) == _native.DPTM_EINVAL and b"aligned" in lib.dptm_layer_last_error()
