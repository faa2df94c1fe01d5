"""The operators of a serving step of many sequences on the GPU where their numbers are few, far apart or infinite, and along paths that ordinary sizes do not take (plain forms in 64 bits: tests/serving_ref.py)."""
import numpy as np
import pytest

import serving_ref as ref
from serving_ref import BF16, F16, F32
from test_gpu_serving import NAN, Step, random_tree, run_adapters
from test_gpu_serving import test_eviction as evicts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from powerserve_amd import hip as h
    return h


def again(step, *names):
    """Arrays of a step that were changed behind its making, to the device."""
    for n in names:
        step.d[n].free()
        step.d[n] = step.ctx.to_device(getattr(step, n))
    step.cache.k, step.cache.v, step.args.q = (step.d[n].ptr for n in ("k", "v", "q"))
    if step.append:
        step.args.k_new, step.args.v_new = step.d["kn"].ptr, step.d["vn"].ptr
    return step


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_new", [1, 4, 60])
def test_a_token_that_takes_almost_all_of_the_weight_and_the_many_that_share_the_rest(ctx, hip, dtype, n_new):
    """An attention sink: one slot 10 to 24 above the others, whose value is zero, so that the result is what thousands of small weights leave."""
    rng = np.random.default_rng(n_new)
    H, G, D = 8, 2, 64
    s = Step(ctx, hip, rng, dtype, H, G, D, 4200, [4100, 900], n_new)
    above = np.array([10.0, 14.0, 16.0, 18.0, 12.0, 17.0, 20.0, 24.0])  # of each query head
    q, kn, vn, k, v = (ref.unpack(getattr(s, n), dtype) for n in ("q", "kn", "vn", "k", "v"))
    q *= 0.3
    q[..., 0] = above / 4 / s.scale
    for x in (k, kn):
        x[..., 0] = 0
    for x in (v, vn):
        x[:] = np.abs(x)
    k[:, 0, 0] = 0
    k[:, 0, 0, :, 0] = 4
    v[:, 0, 0] = 0
    s.q, s.kn, s.vn, s.k, s.v = (ref.pack(x, dtype) for x in (q, kn, vn, k, v))
    again(s, "q", "kn", "vn", "k", "v").run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new", [1, 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_whose_steps_are_coarse(ctx, hip, dtype, n_new, sign):
    """Scores of millions, a float's steps an eighth to a half: no weight passes its type's largest number."""
    rng = np.random.default_rng(n_new)
    s = Step(ctx, hip, rng, dtype, 8, 2, 64, 500, [400, 60, 0], n_new, weights=False)
    s.q, s.k, s.kn = (ref.pack(np.abs(ref.unpack(x, dtype)) * y, dtype) for x, y in ((s.q, sign * 400), (s.k, 30), (s.kn, 30)))  # (one sign, so that none is near zero)
    s.args.scale = s.scale = 8.0
    again(s, "q", "k", "kn").run()
    assert np.isfinite(ref.unpack(s.d["out"].numpy(), dtype)).all()
    s.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new,n_kv", [(1, [40, 1, 3000]), (6, [40, 5, 3000]), (60, [40, 9, 3000])])
def test_infinite_values_of_held_slots(ctx, hip, dtype, n_new, n_kv):
    """A value that is infinite is that in the result, whether its slot is held or new; two of different signs, or a NaN, are NaN; where one slot alone is seen too."""
    rng = np.random.default_rng(n_new)
    s = Step(ctx, hip, rng, dtype, 8, 2, 64, 3100, n_kv, n_new, weights=False)
    v, vn = ref.unpack(s.v, dtype), ref.unpack(s.vn, dtype)
    for i, n in enumerate(n_kv):
        for e, x in ((5, np.inf), (6, -np.inf), (7, NAN), (8, np.inf)):
            v[i, n // 2, 0, :, e] = x
        v[i, n - 1, 0, :, 8] = -np.inf if n > 1 else np.inf
    vn[:, -1, :, 9] = np.inf  # beside a new one
    s.v, s.vn = ref.pack(v, dtype), ref.pack(vn, dtype)
    again(s, "v", "vn").run().check()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_single_slot_of_infinite_values(ctx, hip, dtype):
    rng = np.random.default_rng(1)
    s = Step(ctx, hip, rng, dtype, 4, 2, 64, 40, [1, 1], 1, tree=np.zeros((2, 1, 1)), weights=False)
    v = ref.unpack(s.v, dtype)
    v[0, 0, 0, :, ::2] = np.inf
    v[1, 0, 0, :, 1::2] = -np.inf
    s.v = ref.pack(v, dtype)
    again(s, "v").run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new", [1, 60])
def test_infinite_values_of_the_smallest_weights(ctx, hip, dtype, n_new):
    """Slots 100 to 200 below another one, whose weights no float holds, in its block, in its part and in others: infinite is what an infinite value is times any weight."""
    rng = np.random.default_rng(n_new)
    D = 64
    s = Step(ctx, hip, rng, dtype, 4, 2, D, 3100, [3000, 200, 3000], n_new, weights=False)
    q, kn, k, v = (ref.unpack(getattr(s, n), dtype) for n in ("q", "kn", "k", "v"))
    q[..., 0] = 30
    kn[..., 0] = k[..., 0] = 0
    for i, at in enumerate((10, 150, 2900)):
        k[i, at, 0, :, 0] = (100, 150, 200)[i] / 30 / s.scale
    for i, n in enumerate(s.n0):
        for e, j in enumerate((0, 11, 40, 120, 199, 2000)):
            if j < n:
                v[i, j, 0, :, e] = np.inf if e % 2 else -np.inf
    s.q, s.kn, s.k, s.v = (ref.pack(x, dtype) for x in (q, kn, k, v))
    again(s, "q", "kn", "k", "v").run().check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_new,as_tree", [(9, False), (24, True), (150, False)])
def test_many_rows_are_as_exact_as_few(ctx, hip, dtype, n_new, as_tree):
    """A drafted token's result does not depend on how many are drafted with it: rounding a weight is 2^-16 of it at most, whatever the number of rows.  (Few slots, so that the values of a row do not even the roundings out.)"""
    rng = np.random.default_rng(n_new)
    H, G, D, S = 8, 2, 64, 6
    tree = random_tree(rng, S, n_new) if as_tree else None
    s = Step(ctx, hip, rng, dtype, H, G, D, 400, [0, 1, 2, 5, 3, 200], n_new, tree=tree, weights=False).run()
    out, K, V, q, kn, vn = (ref.unpack(x, dtype) for x in (s.d["out"].numpy(), s.k, s.v, s.q, s.kn, s.vn))
    for i in range(S):
        n0 = int(s.n0[i])
        K[i, n0:n0 + n_new, 0], V[i, n0:n0 + n_new, 0] = kn[i], vn[i]
        want, _, size, far = ref.attend(q[i], K[i, :, 0], V[i, :, 0], n0, n_new, s.scale, None if tree is None else tree[i])
        # as in Step.check; the weights as two numbers: 2^-16
        rel = 2 * (D + 4) * 2.0**-24 * far + 2 * 2.0**-22 + (n0 + n_new + 64) * 2.0**-23 + 2.0**-16
        bound = rel * size + ref.HALF_STEP[dtype] * (np.abs(want) + rel * size) + ref.TINY[dtype]
        err = np.abs(out[i] - want)
        assert (err <= bound).all(), (i, float((err / bound).max()))
    s.free()


@pytest.mark.parametrize("n_new", [1, 60])
def test_small_products_of_a_score_are_not_all_lost_beside_a_large_one(ctx, hip, n_new):
    """fp32: a score of 1 and 63 times 2^-26 is a sum of even and one of odd numbers, of which one has the 1: the other's 32 small products add up exactly and their sum does to the 1, so that 31 of them at most are
    lost.  Times 2^20, beside a slot whose score is 1: the quotient of the two weights is e^(63/64), the exponent 31/64 too small at most."""
    rng = np.random.default_rng(2)
    s = Step(ctx, hip, rng, F32, 4, 2, 64, 80, [2], n_new, tree=np.zeros((1, n_new, n_new)))
    s.q[...] = 1
    s.k[0, :2] = 0
    s.k[0, 0] = 2.0**-26
    s.k[0, :2, 0, :, 0] = 1
    s.weight[...] = 0
    again(s, "q", "k")
    s.d["weight"].free()
    s.d["weight"] = ctx.to_device(s.weight)
    s.cache.weight = s.d["weight"].ptr
    s.args.scale = 2.0**20
    w = s.run().d["weight_out"].numpy().astype(np.float64)[0, :, :2]
    got = np.log(w[:, 0] / w[:, 1])
    assert (got >= 32 / 64 - 1e-5).all() and (got <= 63 / 64 + 1e-5).all(), got  # (1e-5: e^x to 2^-22, sums of at most 120 weights)
    s.free()


# ---------------------------------------------------------------------------------------------------------------------------- paths that ordinary sizes do not take
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S,G,n_ctx,n_new", [(64, 8, 256, 12), (32, 8, 500, 40), (128, 4, 200, 9)])
def test_weights_of_portions_of_many_sequences(ctx, hip, dtype, S, G, n_ctx, n_new):
    """33 to 256 rows a kv head, slots enough to fill the chip: a work-group has all rows of its slots, of which the causal mask leaves some out"""
    rng = np.random.default_rng(S)
    n_kv = rng.integers(0, n_ctx + 1, S)
    Step(ctx, hip, rng, dtype, 4 * G, G, 32, n_ctx, n_kv, n_new, count=np.where(np.arange(S) % 7 == 6, 0, rng.integers(1, n_new + 1, S))).run().check()


@pytest.mark.parametrize("dtype,dim", [(F32, 8), (BF16, 16)])
@pytest.mark.parametrize("n_ctx,n_kv,keep,recent,first", [(32768, [32768, 16384, 16385, 20000], 2048, 300, 4), (20001, [20001, 17000], 16390, 16000, 0), (32767, [32767, 30000], 30001, 1, 1), (16400, [16399], 1, 0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_with_keys_in_lds_and_more_slots_than_are_loaded_at_once(ctx, hip, dtype, dim, n_ctx, n_kv, keep, recent, first, in_place):
    evicts(ctx, hip, dtype, dim, n_ctx, n_kv, keep, recent, first, in_place)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,N,slots", [(3000, 1000, 2999), (3000, 997, 3500), (4200, 601, 4300)])
def test_adapters_of_more_than_256_columns_a_work_group(ctx, hip, dtype, T, N, slots):
    rng = np.random.default_rng(N)
    run_adapters(ctx, hip, rng, dtype, T, N, 24, [2, 1] * (slots // 2), rng.integers(-1, slots + 2, T))
