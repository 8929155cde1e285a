"""Layer operators on the GPU where values are what goes wrong: non-finite operands of pairs that do not count, rows of NaN, gradients
far from one.  Expected values are the float64 restatement's (oracle/layers_ref.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from deepptmpred_amd import layers  # noqa: E402
from oracle import layers_ref as R  # noqa: E402
from test_gpu_layers import host, tensor, within  # noqa: E402

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
