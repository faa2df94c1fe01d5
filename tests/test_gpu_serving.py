"""The operators of a serving step of many sequences on the GPU against plain forms in 64 bits (tests/serving_ref.py)."""
import ctypes as C
import math

import numpy as np
import pytest

import serving_ref as ref
from serving_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(scope="module")
def hip():
    from powerserve_amd import hip as h
    return h


class Step:
    """Caches, new tokens and their places on the device; slots that nobody holds are NaN, results start as a number that nothing computes."""

    def __init__(self, ctx, hip, rng, dtype, heads, kv_heads, dim, n_ctx, n_kv, n_new, count=None, tree=None, weights=True, append=True, spread=1, offset=0, qscale=1.5):
        self.ctx, self.hip, self.dtype, self.dim, self.heads, self.kv_heads, self.n_ctx, self.n_new = ctx, hip, dtype, dim, heads, kv_heads, n_ctx, n_new
        S = self.S = len(n_kv)
        self.n0, self.cnt = ref.lengths(n_kv, count, n_ctx, n_new)
        self.scale, self.tree, self.append = 1 / math.sqrt(dim), tree, append
        p = lambda x: ref.pack(x, dtype)  # noqa: E731
        self.q, self.kn, self.vn = p(qscale * rng.standard_normal((S, n_new, heads, dim))), p(rng.standard_normal((S, n_new, kv_heads, dim))), p(rng.standard_normal((S, n_new, kv_heads, dim)))
        k, v = np.full((S, n_ctx, spread, kv_heads, dim), NAN), np.full((S, n_ctx, spread, kv_heads, dim), NAN)
        for s in range(S):
            k[s, :self.n0[s], offset], v[s, :self.n0[s], offset] = rng.standard_normal((2, self.n0[s], kv_heads, dim))
        self.k, self.v, self.layer = p(k), p(v), offset
        if not append:
            for s in range(S):
                e = self.n0[s] + self.cnt[s]
                self.k[s, self.n0[s]:e, offset], self.v[s, self.n0[s]:e, offset] = self.kn[s, :self.cnt[s]], self.vn[s, :self.cnt[s]]
        self.weight = (rng.random((S, kv_heads, n_ctx)) * 3).astype(np.float32) if weights else None
        self.pos = np.tile(np.arange(n_ctx, dtype=np.int32), (S, kv_heads, 1))
        up = ctx.to_device
        self.d = {n: up(getattr(self, n)) for n in ("q", "k", "v", "kn", "vn", "pos")}
        self.d["n_kv"], self.d["out"] = up(np.asarray(n_kv, dtype=np.int32)), up(p(np.full(self.q.shape, 77.0)))
        self.d["count"] = up(np.asarray(count, dtype=np.int32)) if count is not None else None
        self.d["tree"] = up(np.asarray(tree, dtype=np.uint8)) if tree is not None else None
        if weights:
            self.d["weight"], self.d["weight_out"] = up(self.weight), up(np.full(self.weight.shape, -5.0, dtype=np.float32))
        item = self.k.itemsize
        row = spread * kv_heads * dim
        at = offset * kv_heads * dim * item
        self.cache = hip.kv_cache(dtype, self.d["k"].ptr + at, self.d["v"].ptr + at, self.d["n_kv"], S, n_ctx, kv_heads, dim, pos=self.d["pos"], weight=self.d.get("weight"), strides=(n_ctx * row, row, dim))
        self.args = hip.cache_attn_args(self.d["q"], self.d["out"], heads, n_new, self.scale, k_new=self.d["kn"] if append else None, v_new=self.d["vn"] if append else None, count=self.d["count"],
                                        tree=self.d["tree"], weight_out=self.d.get("weight_out"))
        self.need = ctx.cache_attn_workspace(self.cache, self.args)
        self.space = ctx.empty(max(self.need, 16), np.uint8)

    def run(self):
        self.ctx.cache_attn(self.cache, self.args, self.space, self.need)
        return self

    def free(self):
        for x in list(self.d.values()) + [self.space]:
            if x is not None:
                x.free()

    def check(self):
        out, k, v = (ref.unpack(self.d[n].numpy(), self.dtype) for n in ("out", "k", "v"))
        w = self.d["weight_out"].numpy() if self.weight is not None else None
        K, V = ref.unpack(self.k, self.dtype), ref.unpack(self.v, self.dtype)
        q, kn, vn = (ref.unpack(x, self.dtype) for x in (self.q, self.kn, self.vn))
        for s in range(self.S):
            n0, cnt = int(self.n0[s]), int(self.cnt[s])
            K[s, n0:n0 + cnt, self.layer], V[s, n0:n0 + cnt, self.layer] = kn[s, :cnt], vn[s, :cnt]
            want, weight, size, far = ref.attend(q[s], K[s, :, self.layer], V[s, :, self.layer], n0, cnt, self.scale, None if self.tree is None else np.asarray(self.tree)[s])
            # a score is a sum of dim products, rounded dim times at most, and scaled (twice: scale and log2 e); e^x of the hardware and of a difference of two such numbers: 2^-22 of it, and what
            # its argument is off by; sums of weights and of products over n slots, in parts: n + 64 roundings; 16-bit weights as two numbers: 2^-16, of more than 32 rows as one: its rounding; then the result's own rounding
            score = (self.dim + 4) * 2.0**-24 * far
            rel = 2 * score + 2 * 2.0**-22 + (n0 + cnt + 64) * 2.0**-23 + (0 if self.dtype == F32 else 2.0**-16 if self.n_new * self.heads <= 32 * self.kv_heads else ref.HALF_STEP[self.dtype])
            bound = rel * size + ref.HALF_STEP[self.dtype] * (np.abs(want) + rel * size) + ref.TINY[self.dtype]
            fine = np.isfinite(want)
            assert np.array_equal(np.isnan(out[s, :cnt]), np.isnan(want)) and np.array_equal(out[s, :cnt][~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
            err = np.abs(out[s, :cnt] - want)
            assert (err[fine] <= bound[fine]).all(), (s, float((err - bound)[fine].max()), float(err[fine].max()))
            assert (out[s, cnt:] == 77.0).all()
            if w is not None:
                held = weight.copy()
                held[:, :n0] += self.weight[s, :, :n0].astype(np.float64)
                rows = cnt * self.heads // self.kv_heads
                tol = (2 * score + 2 * 2.0**-22 + (n0 + 2 * cnt + 64 + rows) * 2.0**-23) * weight + 2.0**-23 * held
                assert (np.abs(w[s, :, :n0 + cnt] - held) <= tol).all(), float((np.abs(w[s, :, :n0 + cnt] - held) - tol).max())
                assert (w[s, :, n0 + cnt:] == -5.0).all()
        assert np.array_equal(k, K, equal_nan=True) and np.array_equal(v, V, equal_nan=True)
        self.free()


def random_tree(rng, S, T):
    tree = np.zeros((S, T, T), dtype=np.uint8)
    for s in range(S):
        for t in range(T):
            if t and rng.random() < 0.85:
                tree[s, t] = tree[s, rng.integers(0, t)]
            tree[s, t, t] = 1
    return tree


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (32, 8, 128), (3, 3, 96), (8, 1, 8), (5, 5, 40)])
def test_single_tokens_of_sequences_of_all_lengths(ctx, hip, dtype, heads, kv_heads, dim):
    rng = np.random.default_rng(heads + dim + dtype)
    Step(ctx, hip, rng, dtype, heads, kv_heads, dim, 1100, [0, 1, 31, 32, 33, 127, 128, 129, 700, 1099, 1100, 1], 1).run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new,heads,kv_heads,dim", [(2, 14, 2, 64), (9, 32, 8, 128), (24, 8, 2, 128), (70, 4, 4, 64), (150, 6, 2, 96), (3, 33, 1, 64), (129, 8, 2, 128), (300, 3, 1, 40)])
@pytest.mark.parametrize("weights", [True, False])
def test_portions_behind_caches(ctx, hip, dtype, n_new, heads, kv_heads, dim, weights):
    rng = np.random.default_rng(n_new + dim + dtype)
    Step(ctx, hip, rng, dtype, heads, kv_heads, dim, 600, [0, 1, 130, 450, 600, 597], n_new, count=[n_new, n_new - 1, 0, n_new, n_new, 5], weights=weights).run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new,heads,kv_heads,dim", [(5, 14, 2, 64), (24, 32, 8, 128), (40, 6, 2, 96)])
def test_trees_of_drafted_tokens(ctx, hip, dtype, n_new, heads, kv_heads, dim):
    rng = np.random.default_rng(n_new + dim + dtype)
    tree = random_tree(rng, 4, n_new)
    tree[1, n_new // 2] = 0  # a token that sees nothing new
    tree[3, 0] = 0           # and one that sees nothing at all
    Step(ctx, hip, rng, dtype, heads, kv_heads, dim, 400, [17, 0, 333, 0], n_new, count=[n_new, n_new, n_new - 2, n_new], tree=tree).run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_that_are_there_already_and_layers_between_each_other(ctx, hip, dtype):
    rng = np.random.default_rng(3)
    Step(ctx, hip, rng, dtype, 8, 2, 64, 300, [5, 250, 0], 7, append=False, spread=3, offset=1).run().check()
    Step(ctx, hip, rng, dtype, 8, 2, 128, 300, [5, 250, 0], 1, spread=2, offset=1).run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new", [6, 60])
def test_odd_numbers_reach_only_those_who_see_them(ctx, hip, dtype, n_new):
    """NaN and infinities in keys and values of drafted tokens: a token that sees them has them, the others do not."""
    rng = np.random.default_rng(n_new)
    s = Step(ctx, hip, rng, dtype, 4, 2, 64, 300, [40, 0], n_new, weights=False)
    s.vn[:, 3, :, 5] = ref.pack(np.inf, dtype)
    s.vn[:, 4, :, 6] = ref.pack(NAN, dtype)
    s.kn[:, 5, :, 7] = ref.pack(NAN, dtype)
    s.d["kn"].free(), s.d["vn"].free()
    s.d["kn"], s.d["vn"] = ctx.to_device(s.kn), ctx.to_device(s.vn)
    s.args.k_new, s.args.v_new = s.d["kn"].ptr, s.d["vn"].ptr
    s.run().check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_repeated_step_changes_nothing(ctx, hip, dtype):
    rng = np.random.default_rng(5)
    s = Step(ctx, hip, rng, dtype, 32, 8, 128, 900, [800, 3, 410], 4)
    first = s.run().d["out"].numpy(), s.d["weight_out"].numpy()
    for _ in range(3):
        again = s.run().d["out"].numpy(), s.d["weight_out"].numpy()
        assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(first, again))
    s.check()


def test_weights_in_place_and_positions_of_new_tokens(ctx, hip):
    rng = np.random.default_rng(6)
    s = Step(ctx, hip, rng, F16, 8, 2, 64, 200, [150, 0, 199], 3, count=[3, 2, 3])
    pos_new = ctx.to_device(np.arange(1000, 1009, dtype=np.int32).reshape(3, 3))
    s.args.pos_new = pos_new.ptr
    before = s.weight.copy()
    want = s.run().d["weight_out"].numpy()
    s.args.weight_out = s.d["weight"].ptr
    got = s.run().d["weight"].numpy()
    pos = s.d["pos"].numpy()
    for i, (n0, cnt) in enumerate(zip(s.n0, s.cnt)):
        e = n0 + cnt
        assert np.array_equal(got[i, :, :e], want[i, :, :e]) and np.array_equal(got[i, :, e:], before[i, :, e:])
        assert (pos[i, :, n0:e] == 1000 + 3 * i + np.arange(cnt)).all() and (pos[i, :, :n0] == np.arange(n0)).all() and (pos[i, :, e:] == np.arange(e, 200)).all()
    s.free()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_an_accepted_path_becomes_part_of_the_cache(ctx, hip, dtype):
    rng = np.random.default_rng(7)
    s = Step(ctx, hip, rng, dtype, 4, 2, 40, 60, [20, 0, 55, 58, 7], 6, append=False)
    take = np.array([[0, 2, 5, 0], [1, 2, 3, 4], [0, 4, 0, 0], [1, 2, 0, 0], [0, 0, 3, 4]], dtype=np.int32)
    count = np.array([3, 4, 2, 2, 4], dtype=np.int32)
    k, v, pos, w = s.k.copy(), s.v.copy(), s.pos.copy(), s.weight.copy()
    n_want = []
    for i in range(5):
        last, n = -1, 0
        for t in take[i, :count[i]]:
            if t <= last or s.n0[i] + t >= 60:
                break
            last = t
            for x in (k[i], v[i]):
                x[s.n0[i] + n] = x[s.n0[i] + t]
            for x in (pos[i], w[i]):
                x[:, s.n0[i] + n] = x[:, s.n0[i] + t]
            n += 1
        n_want.append(s.n0[i] + n)
    dt, dc = ctx.to_device(take), ctx.to_device(count)
    ctx.cache_advance(s.cache, dc, dt, 4)
    assert np.array_equal(s.d["n_kv"].numpy(), n_want)
    for name, want in (("k", k), ("v", v), ("pos", pos), ("weight", w)):
        assert np.array_equal(s.d[name].numpy().view(np.uint8), want.view(np.uint8)), name
    ctx.cache_advance(s.cache, ctx.to_device(np.array([1, 60, 9, -3, 2], dtype=np.int32)))
    assert np.array_equal(s.d["n_kv"].numpy(), np.clip(np.array(n_want) + [1, 60, 9, 0, 2], 0, 60))
    s.free()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new", [1, 5, 70])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1e-3])
def test_scales_of_every_kind(ctx, hip, dtype, n_new, scale):
    rng = np.random.default_rng(n_new)
    s = Step(ctx, hip, rng, dtype, 6, 2, 64, 500, [3, 0, 411], n_new)
    s.args.scale = s.scale = float(np.float32(scale))
    s.run().check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_new,heads,kv_heads,dim", [(7, 32, 8, 128), (5, 8, 2, 128), (8, 4, 1, 88), (17, 3, 3, 64), (1, 20, 1, 128), (32, 1, 1, 16), (33, 1, 1, 128)])
@pytest.mark.parametrize("as_tree", [False, True])
def test_two_tiles_of_rows(ctx, hip, dtype, n_new, heads, kv_heads, dim, as_tree):
    rng = np.random.default_rng(n_new + dim)
    Step(ctx, hip, rng, dtype, heads, kv_heads, dim, 700, [0, 640, 129], n_new, tree=random_tree(rng, 3, n_new) if as_tree else None).run().check()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n_new", [2, 3, 4, 6])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (40, 2)])
def test_small_trees_of_any_bytes(ctx, hip, dtype, n_new, heads, kv_heads):
    """rows of fewer than four bytes, and bytes that are not 0 and not 1"""
    rng = np.random.default_rng(n_new)
    tree = random_tree(rng, 5, n_new) * rng.choice(np.array([1, 2, 127, 128, 255], dtype=np.uint8), (5, n_new, n_new))
    Step(ctx, hip, rng, dtype, heads, kv_heads, 64, 400, [0, 61, 399, 30, 254], n_new, count=[n_new, n_new - 1, n_new, 1, n_new], tree=tree).run().check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S", [255, 256, 257, 300])
def test_many_sequences(ctx, hip, dtype, S):
    rng = np.random.default_rng(S)
    Step(ctx, hip, rng, dtype, 4, 2, 64, 300, rng.integers(0, 300, S), 1).run().check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S", [2, 61, 256, 257])
def test_drafted_tokens_of_many_sequences(ctx, hip, dtype, S):
    """more than 32 rows each, lengths far apart, some without a token"""
    rng = np.random.default_rng(S)
    n_kv = (1090 * rng.random(S) ** 3).astype(int)
    n_kv[0] = 1091
    Step(ctx, hip, rng, dtype, 8, 2, 32, 1100, n_kv, 9, count=np.where(np.arange(S) % 5 == 4, 0, 9), tree=random_tree(rng, S, 9)).run().check()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n_new", [1, 40])
def test_one_long_sequence_and_among_short_ones(ctx, hip, dtype, n_new):
    rng = np.random.default_rng(9)
    Step(ctx, hip, rng, dtype, 2, 1, 64, 40000, [39900], n_new).run().check()
    Step(ctx, hip, rng, dtype, 2, 1, 64, 20000, [0, 19900, 3], n_new).run().check()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n_new", [2, 50])
def test_other_layouts_give_the_same_bits(ctx, hip, dtype, n_new):
    """Heads before slots, rows of q, out, k_new and v_new with something between them, a workspace full of ones, another context: the same result to the bit, and nothing between the rows is touched."""
    rng = np.random.default_rng(n_new)
    S, H, G, D, n_ctx, pad = 3, 8, 2, 72, 400, 24
    s = Step(ctx, hip, rng, dtype, H, G, D, n_ctx, [350, 0, 77], n_new)
    s.run()
    want = [s.d[n].numpy() for n in ("out", "weight_out", "k", "v")]
    other = hip.Ctx(0)
    kt, vt = (other.to_device(np.ascontiguousarray(x[:, :, 0].transpose(0, 2, 1, 3))) for x in (s.k, s.v))

    def wider(x):
        y = np.full((S, n_new + 1, x.shape[2] * D + pad), 3, dtype=x.dtype)
        y[:, :n_new, :x.shape[2] * D] = x.reshape(S, n_new, -1)
        return y

    ow = wider(s.d["out"].numpy() * 0 + ref.pack(77.0, dtype))
    dev = [other.to_device(x) for x in (wider(s.q), wider(s.kn), wider(s.vn), ow)]
    n_kv, w, w_out = other.to_device(np.array([350, 0, 77], dtype=np.int32)), other.to_device(s.weight), other.to_device(np.full(s.weight.shape, -5.0, dtype=np.float32))
    cache = hip.kv_cache(dtype, kt, vt, n_kv, S, n_ctx, G, D, weight=w, strides=(G * n_ctx * D, D, n_ctx * D))
    q_row, n_row = H * D + pad, G * D + pad
    args = hip.cache_attn_args(dev[0], dev[3], H, n_new, s.scale, k_new=dev[1], v_new=dev[2], weight_out=w_out,
                               strides=((n_new + 1) * q_row, q_row, (n_new + 1) * q_row, q_row, (n_new + 1) * n_row, n_row))
    need = other.cache_attn_workspace(cache, args)
    space = other.to_device(np.full(need, 255, dtype=np.uint8))
    other.cache_attn(cache, args, space, need)
    got = dev[3].numpy()
    same = lambda a, b: np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))  # noqa: E731
    assert same(got[:, :n_new, :H * D].reshape(S, n_new, H, D), want[0])
    assert (got[:, n_new:] == ow[:, n_new:]).all() and (got[:, :, H * D:] == ow[:, :, H * D:]).all()
    assert same(w_out.numpy(), want[1]) and same(kt.numpy().transpose(0, 2, 1, 3), want[2][:, :, 0]) and same(vt.numpy().transpose(0, 2, 1, 3), want[3][:, :, 0])
    for x in dev + [kt, vt, n_kv, w, w_out, space]:
        x.free()
    s.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_new", [1, 50])
def test_offsets_past_32_bits(ctx, hip, dtype, n_new):
    """Slots 8 MB apart, 600 of them, a step with eviction: the bits of the same slots one behind the other."""
    rng = np.random.default_rng(n_new)
    G, D, n_ctx, n0, keep = 2, 64, 620, 560, 400
    s = Step(ctx, hip, rng, dtype, 4, G, D, n_ctx, [n0], n_new)
    item, step = s.k.itemsize, 8 << 20
    far = [ctx.empty((n_ctx * step,), np.uint8) for _ in range(2)]
    for x, y in zip(far, (s.k, s.v)):
        for j in range(n0):
            row = np.ascontiguousarray(y[0, j, 0])
            ctx.check(ctx.L.ps_hip_memcpy_h2d(ctx.h, x.ptr + j * step, row.ctypes.data_as(C.c_void_p), row.nbytes))
    got = []
    for k, v, strides in ((s.d["k"].ptr, s.d["v"].ptr, (n_ctx * G * D, G * D, D)), (far[0].ptr, far[1].ptr, (n_ctx * step // item, step // item, D))):
        n_kv, w, pos, one = ctx.to_device(np.array([n0], dtype=np.int32)), ctx.to_device(s.weight), ctx.to_device(s.pos), ctx.to_device(np.array([n_new], dtype=np.int32))
        cache = hip.kv_cache(dtype, k, v, n_kv, 1, n_ctx, G, D, pos=pos, weight=w, strides=strides)
        args, evict = hip.cache_attn_args(s.d["q"], s.d["out"], 4, n_new, s.scale, k_new=s.d["kn"], v_new=s.d["vn"], weight_out=w), hip.cache_evict_args(keep, 30, 2)
        need = [ctx.cache_attn_workspace(cache, args), ctx.cache_evict_workspace(cache, evict)]
        space = [ctx.empty(b, np.uint8) for b in need]
        ctx.cache_attn(cache, args, space[0], need[0])
        ctx.cache_advance(cache, one)
        ctx.cache_evict(cache, evict, space[1], need[1])
        rows = np.empty((2, n0 + n_new, G * D), dtype=s.k.dtype)
        for i, p in enumerate((k, v)):
            for j in range(n0 + n_new):
                ctx.check(ctx.L.ps_hip_memcpy_d2h(ctx.h, rows[i, j].ctypes.data_as(C.c_void_p), p + j * strides[1] * item, G * D * item))
        got.append([s.d["out"].numpy(), w.numpy(), pos.numpy(), n_kv.numpy(), rows])
        for x in [n_kv, w, pos, one] + space:
            x.free()
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    assert got[0][3][0] == keep
    for x in far:
        x.free()
    s.free()


# ---------------------------------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("dtype,dim", [(F32, 8), (F16, 128), (BF16, 40)])
@pytest.mark.parametrize("n_ctx,n_kv,keep,recent,first", [(300, [300, 0, 1, 65, 64, 299], 64, 16, 4), (70, [70, 69, 68], 69, 69, 0), (5000, [5000, 1025, 1024, 4097], 1024, 500, 0),
                                                          (40, [40, 1, 2], 1, 0, 1), (40000, [40000, 33000], 20000, 7, 3), (100, [100, 300, -4], 99, 3, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction(ctx, hip, dtype, dim, n_ctx, n_kv, keep, recent, first, in_place):
    rng = np.random.default_rng(n_ctx + dim)
    S, G = len(n_kv), 2
    k, v = (ref.pack(rng.standard_normal((S, n_ctx, G, dim)), dtype) for _ in range(2))
    w = np.maximum(rng.standard_normal((S, G, n_ctx)) - 0.5, 0).astype(np.float32).round(2)  # many equal ones
    w[0, 0, ::7] = np.nan
    w[0, 1, :] = 1.0
    w[-1, 0, ::3] = np.inf
    pos = np.argsort(rng.random((S, G, n_ctx)), -1).astype(np.int32)
    d = {n: ctx.to_device(x) for n, x in (("k", k), ("v", v), ("w", w), ("pos", pos), ("n", np.asarray(n_kv, dtype=np.int32)))}
    cache = hip.kv_cache(dtype, d["k"], d["v"], d["n"], S, n_ctx, G, dim, pos=d["pos"], weight=d["w"])
    if not in_place:
        d["w2"], d["pos2"], d["n2"] = ctx.to_device(np.full_like(w, -3)), ctx.to_device(np.full_like(pos, -3)), ctx.to_device(np.full(S, -3, dtype=np.int32))
    args = hip.cache_evict_args(keep, recent, first) if in_place else hip.cache_evict_args(keep, recent, first, weight_out=d["w2"], pos_out=d["pos2"], n_kv_out=d["n2"])
    need = ctx.cache_evict_workspace(cache, args)
    space = ctx.empty(max(16, need), np.uint8)
    for _ in range(1 if in_place else 3):
        ctx.cache_evict(cache, args, space, need)
    got = {n: x.numpy() for n, x in d.items()}
    names = ("w", "pos", "n") if in_place else ("w2", "pos2", "n2")
    for s in range(S):
        n = min(max(n_kv[s], 0), n_ctx)
        for g in range(G):
            take = ref.evict(n, keep, recent, first, w[s, g], pos[s, g]) if n > keep else np.arange(n)
            m = len(take)
            assert np.array_equal(got[names[0]][s, g, :m], w[s, g, take], equal_nan=True) and np.array_equal(got[names[1]][s, g, :m], pos[s, g, take])
            for x, y in (("k", k), ("v", v)):
                assert np.array_equal(got[x][s, :m, g], y[s, take, g]) and np.array_equal(got[x][s, m:, g], y[s, m:, g])
            if in_place:
                assert np.array_equal(got["w"][s, g, m:], w[s, g, m:], equal_nan=True) and np.array_equal(got["pos"][s, g, m:], pos[s, g, m:])
            else:
                assert (got["w2"][s, g, m:] == -3).all() and (got["pos2"][s, g, m:] == -3).all()
        assert got[names[2]][s] == min(n, keep)
    for x in list(d.values()) + [space]:
        x.free()


def test_eviction_takes_the_two_zeros_as_equal(ctx, hip):
    n, keep, dim = 80, 30, 8
    k, v = np.random.default_rng(8).standard_normal((2, 1, n, 1, dim)).astype(np.float32)
    w = np.zeros((1, 1, n), dtype=np.float32)
    w[0, 0, :40:3] = -0.0  # below it a slot at the end would stay for one of these
    pos = np.arange(n, dtype=np.int32).reshape(1, 1, n)
    d = [ctx.to_device(x) for x in (k, v, np.array([n], dtype=np.int32), pos, w)]
    cache, args = hip.kv_cache(F32, d[0], d[1], d[2], 1, n, 1, dim, pos=d[3], weight=d[4]), hip.cache_evict_args(keep)
    need = ctx.cache_evict_workspace(cache, args)
    space = ctx.empty(need, np.uint8)
    ctx.cache_evict(cache, args, space, need)
    assert np.array_equal(d[0].numpy()[0, :keep], k[0, :keep]) and np.array_equal(d[3].numpy()[0, 0, :keep], np.arange(keep)) and d[2].numpy()[0] == keep
    for x in d + [space]:
        x.free()


# ---------------------------------------------------------------------------------------------------------------------------- sampling
def run_sample(ctx, hip, logits, dtype, rows_settings, stride=None):
    """logits: the type's bits [rows, n]; rows_settings: (temperature, top_k, top_p, min_p, u) arrays or None"""
    R, n = logits.shape
    stride = stride or n
    padded = np.zeros((R, stride), dtype=logits.dtype)
    padded[:, :n] = logits
    kinds = (np.float32, np.int32, np.float32, np.float32, np.float32)
    dev = [None if x is None else ctx.to_device(np.asarray(x, dtype=k)) for x, k in zip(rows_settings, kinds)]
    dl, ids, prob = ctx.to_device(padded), ctx.empty((R,), np.int32), ctx.empty((R,), np.float32)
    need = ctx.sample_workspace(n, R)
    space = ctx.empty(max(16, need), np.uint8)
    p = hip.sample_params(temperature=dev[0], top_k=dev[1], top_p=dev[2], min_p=dev[3], u=dev[4])
    ctx.sample(dl, n, R, p, ids, prob=prob, dtype=dtype, stride=stride, space=space, space_bytes=need)
    got = ids.numpy(), prob.numpy()
    ctx.sample(dl, n, R, p, ids, dtype=dtype, stride=stride, space=space, space_bytes=need)
    assert np.array_equal(ids.numpy(), got[0])
    for x in [dl, ids, prob, space] + [d for d in dev if d is not None]:
        x.free()
    return got


def check_sample(ctx, hip, logits, dtype, settings, stride=None):
    ids, prob = run_sample(ctx, hip, logits, dtype, settings, stride)
    wide = ref.unpack(logits, dtype)
    off = (1.0, 0, 1.0, 0.0)
    for r in range(len(ids)):
        row = [off[i] if settings[i] is None else settings[i][r] for i in range(4)] + [settings[4][r]]
        # the numbers as the device has them
        row = [float(np.float32(x)) for x in row]
        want, p, near = ref.sample(wide[r], row[0], int(row[1]), row[2], row[3], row[4])
        # a weight is off by 2^-27 of itself (z in 64 bits; the difference of e^-f from 1, f < 2^-5, in 32 bits: f rounded, two roundings of the last steps, 3 x 2^-24 of at most 2^-5) and by half a
        # multiple of 2^-38 or less: a sum and what it is compared with, 2^-26 of the whole together, or the number is one of those that may answer otherwise
        if near < 2.0**-25:
            continue
        assert ids[r] == want, (r, row, ids[r], want, near)
        # prob: a quotient of two of them, rounded once
        assert abs(prob[r] - p) <= (2.0**-24 + 2.0**-26) * p + 1e-9, (r, prob[r], p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (5, 50), (2, 4096), (7, 4097), (1, 32000), (3, 128256), (150, 999), (300, 5003), (64, 20001)])
def test_sampling_with_all_settings(ctx, hip, dtype, rows, n):
    rng = np.random.default_rng(n + dtype)
    logits = ref.pack(2.5 * rng.standard_normal((rows, n)) + 8 * rng.random((rows, n)) ** 20, dtype)
    settings = [rng.choice([0.3, 0.8, 1.0, 1.7, 0.0], rows), rng.choice([0, 1, 5, 40, 1000, 30000], rows), rng.choice([1.0, 0.95, 0.5, 0.9, 0.1], rows), rng.choice([0.0, 0.02, 0.3], rows), rng.random(rows)]
    check_sample(ctx, hip, logits, dtype, settings, stride=n + rows % 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(6, 27424), (2, 16385), (1, 8200), (9, 8191), (130, 8193)])
@pytest.mark.parametrize("masked", [0.0, 0.97])
def test_sampling_of_short_parts_and_masked_rows(ctx, hip, dtype, rows, n, masked):
    """parts of a row with fewer numbers than threads, and vocabularies most of which a grammar forbids"""
    rng = np.random.default_rng(n + dtype)
    logits = 2.5 * rng.standard_normal((rows, n))
    logits[rng.random((rows, n)) < masked] = -np.inf
    settings = [rng.choice([0.6, 1.0, 1.3], rows), rng.choice([0, 40, 5000], rows), rng.choice([1.0, 0.9], rows), rng.choice([0.0, 0.01], rows), rng.random(rows)]
    check_sample(ctx, hip, ref.pack(logits, dtype), dtype, settings, stride=n + 1)


@pytest.mark.parametrize("rows", [2, 200])
def test_sampling_without_settings(ctx, hip, rows):
    rng = np.random.default_rng(rows)
    logits = ref.pack(3 * rng.standard_normal((rows, 3001)), F32)
    check_sample(ctx, hip, logits, F32, [None, None, None, None, rng.random(rows)])


@pytest.mark.parametrize("rows", [6, 192])
@pytest.mark.parametrize("n", [9000, 40000])
def test_sampling_where_a_bin_outgrows_the_list(ctx, hip, rows, n):
    """Equal logits, few different ones, temperatures that flatten everything: the walk by digits."""
    rng = np.random.default_rng(n + rows)
    logits = np.zeros((rows, n), dtype=np.float32)
    logits[1::3] = rng.integers(0, 3, (len(logits[1::3]), n)) * 0.25 - 1
    logits[2::3] = rng.standard_normal((len(logits[2::3]), n))
    t = np.where(np.arange(rows) % 3 == 2, rng.choice([1e6, 30.0, 200.0], rows), 1.0)
    settings = [t, rng.choice([0, 5000, 7, 8000], rows), rng.choice([1.0, 0.6, 0.93], rows), np.zeros(rows), rng.random(rows)]
    check_sample(ctx, hip, logits, F32, settings)


@pytest.mark.parametrize("rows", [1, 140])
def test_sampling_at_the_borders(ctx, hip, rows):
    n = 777
    rng = np.random.default_rng(rows)
    base = 2 * rng.standard_normal((rows, n)).astype(np.float32)

    def one(logits, *settings):
        check_sample(ctx, hip, logits, F32, [None if x is None else np.full(rows, x) for x in settings])

    masked = base.copy()
    masked[:, 3:] = -np.inf
    one(masked, 1.0, 0, 1.0, 0.0, 0.999)
    nothing = np.full_like(base, -np.inf)
    nothing[:, 5] = np.nan
    one(nothing, 1.0, 3, 0.5, 0.1, 0.5)
    odd = base.copy()
    odd[:, 7] = np.nan
    odd[:, [9, 11]] = np.inf
    one(odd, 1.0, 0, 1.0, 0.0, 0.7)
    low = base.copy()
    low[:, 4:] = np.finfo(np.float32).min  # a mask of the type's lowest value
    one(low, 1.0, 0, 1.0, 0.0, 1.0)
    one(low, 1.0, 9, 0.9, 0.0, 0.9)
    for u in (0.0, 1.0, -1.0, NAN, 2.0, 0.99999994):
        ids, _ = run_sample(ctx, hip, base, F32, [None, np.full(rows, 10), None, None, np.full(rows, u)])
        want = [ref.sample(base[r], 1.0, 10, 1.0, 0.0, 0.0 if not u > 0 else float(np.float32(u)))[0] for r in range(rows)]
        assert np.array_equal(ids, want), u
    one(base, 1.0, 0, 0.0, 0.0, 0.5)
    one(base, 1.0, 0, 1.0, 2.0, 0.5)
    one(base, -1.0, 0, 0.5, 0.0, 0.5)
    one(base, NAN, 0, 0.5, 0.0, 0.5)
    one(base, 1.0, n + 5, NAN, NAN, 0.25)
    one(base, 1e-30, 0, 1.0, 0.0, 0.99)
    one(np.where(base > 0, np.float32(0.0), np.float32(-0.0)), 1.0, 3, 1.0, 0.0, 0.9)


@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("n", [777, 30000])
def test_sampling_with_settings_at_the_ends_of_their_types(ctx, hip, rows, n):
    rng = np.random.default_rng(n)
    base = 2 * rng.standard_normal((rows, n)).astype(np.float32)
    for settings in ((np.inf, 0, 1.0, 0.0, 0.3), (1e-45, 0, 1.0, 0.0, 0.9), (3e38, 9, 0.7, 0.0, 0.6), (1.0, 2**31 - 1, 1.0, 0.0, 0.4), (1.0, -2**31, 0.999, 0.0, 0.4), (1.0, 1, 1e-40, 1e-40, 0.4),
                     (-0.0, 3, 1.0, 0.0, 0.4), (1.0, 1014, 1.0, 0.0, 0.77), (1.0, 1015, 1.0, 0.0, 0.77), (0.5, 0, -1.0, -1.0, 0.5)):
        check_sample(ctx, hip, base, F32, [np.full(rows, x) for x in settings])
    wide = np.where(base > 0, np.float32(3.4e38), np.float32(-3.4e38))
    check_sample(ctx, hip, wide, F32, [np.full(rows, x) for x in (1.0, 0, 1.0, 0.0, 0.6)])


# ---------------------------------------------------------------------------------------------------------------------------- adapters
def run_adapters(ctx, hip, rng, dtype, T, N, K, ranks, ids, pad=0, in_place=False, base=True):
    down = [ref.pack(rng.standard_normal((r, K)) / math.sqrt(K), BF16) for r in ranks]
    up = [ref.pack(rng.standard_normal((N, r)), BF16) for r in ranks]
    scale = [float(np.float32(0.3 + 0.2 * i)) for i in range(len(ranks))]
    a = hip.Adapters(ctx, N, K, len(ranks) + 1, max(ranks))  # (the last slot stays empty)
    for i, r in enumerate(ranks):
        a.load(i, down[i], up[i], scale[i])
    x = ref.pack(rng.standard_normal((T, K + pad)) * 3, dtype)
    b = rng.standard_normal((T, N + pad)).astype(np.float32)
    dx, db, di = ctx.to_device(x), ctx.to_device(b), ctx.to_device(np.asarray(ids, dtype=np.int32))
    out = db if in_place else ctx.to_device(np.full_like(b, 9))
    need = a.workspace(T)
    space = ctx.empty(max(16, need), np.uint8)
    a.apply(dx, T, di, out, base=db if base else None, dtype=dtype, ldx=K + pad, ldo=N + pad, space=space, space_bytes=need)
    got = out.numpy()
    assert np.array_equal(got[:, N:], b[:, N:] if in_place else np.full((T, pad), 9))
    X, B = ref.unpack(x, dtype)[:, :K], b[:, :N].astype(np.float64)
    if not base:
        B[:] = 0
    for t, i in enumerate(ids):
        if not 0 <= i < len(ranks):
            assert np.array_equal(got[t, :N], B[t].astype(np.float32))
            continue
        d, u = ref.unpack(down[i], BF16), ref.unpack(up[i], BF16)
        want = B[t] + scale[i] * (u @ (d @ X[t]))
        # exact products; K + 16 roundings of the inner sums (in parts), rank of the outer ones, three pieces of x and h (2^-23 of them together), the last multiply-add
        size = scale[i] * (np.abs(u) @ (np.abs(d) @ np.abs(X[t])))
        assert (np.abs(got[t, :N] - want) <= ((K + 3 * ranks[i] + 32) * 2.0**-24 + 2.0**-22) * size + 2.0**-24 * (np.abs(want) + np.abs(B[t]))).all(), (t, i)
    a.close()
    for y in {id(z): z for z in (dx, db, di, out, space)}.values():
        y.free()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,N,K,ranks", [(1, 64, 64, [16]), (4, 2048, 2048, [16, 16, 8]), (33, 300, 520, [1, 7, 64, 33]), (256, 128, 96, [4, 200, 16, 17, 5]), (257, 129, 77, [3, 16]), (700, 1000, 1031, [16, 8, 40]),
                                         (40, 1, 1, [2, 1])])
def test_adapters(ctx, hip, dtype, T, N, K, ranks):
    rng = np.random.default_rng(T + N + K)
    ids = rng.integers(-1, len(ranks) + 1, T)
    ids[T // 2] = 10**6
    run_adapters(ctx, hip, rng, dtype, T, N, K, ranks, ids)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adapters_of_long_runs_strides_and_in_place(ctx, hip, dtype):
    rng = np.random.default_rng(1)
    run_adapters(ctx, hip, rng, dtype, 500, 260, 130, [16, 5], [0] * 243 + [1] * 200 + [-1] * 57, pad=3)
    run_adapters(ctx, hip, rng, dtype, 100, 256, 128, [16, 5], [0] * 60 + [1] * 33 + [-1] * 7, pad=8, in_place=True)
    run_adapters(ctx, hip, rng, dtype, 5, 256, 128, [16, 5], [0, 1, -1, 2, 0], base=False)


def test_many_adapters_of_many_tokens(ctx, hip):
    rng = np.random.default_rng(2)
    run_adapters(ctx, hip, rng, BF16, 1500, 32, 64, [2] * 1100, rng.integers(0, 1100, 1500))


def test_more_adapters_than_the_plan_counts_in_lds(ctx, hip):
    rng = np.random.default_rng(12)
    run_adapters(ctx, hip, rng, F32, 300, 12, 20, [1] * 8300, np.where(rng.random(300) < 0.5, 8299, rng.integers(0, 8301, 300)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [20, 90])
def test_odd_numbers_of_a_token_stay_its_own(ctx, hip, dtype, T):
    """Infinities and NaN in some tokens' x, and the largest numbers: the other tokens of the same adapter have the bits that they have without them."""
    rng = np.random.default_rng(T)
    a = hip.Adapters(ctx, 40, 100, 1, 24)
    a.load(0, ref.pack(rng.standard_normal((24, 100)), BF16), ref.pack(rng.standard_normal((40, 24)), BF16), 0.5)
    x = ref.pack(rng.standard_normal((T, 100)), dtype)
    odd = x.copy()
    odd[[3, 4, 17], [7, 99, 0]] = ref.pack([np.inf, NAN, -np.inf], dtype)
    ids, need = ctx.to_device(np.zeros(T, dtype=np.int32)), a.workspace(T)
    space, out = ctx.empty(need, np.uint8), ctx.empty((T, 40))
    got = []
    for y in (x, odd):
        d = ctx.to_device(y)
        a.apply(d, T, ids, out, dtype=dtype, space=space, space_bytes=need)
        got.append(out.numpy())
        d.free()
    others = np.setdiff1d(np.arange(T), [3, 4, 17])
    assert np.array_equal(got[0][others].view(np.uint32), got[1][others].view(np.uint32)) and not np.isfinite(got[1][[3, 4, 17]]).any() and np.isfinite(got[0]).all()
    a.close()
    for y in (ids, space, out):
        y.free()


def test_adapter_slots_change(ctx, hip):
    rng = np.random.default_rng(4)
    a = hip.Adapters(ctx, 32, 64, 2, 16)
    x, b = rng.standard_normal((3, 64)).astype(np.float32), rng.standard_normal((3, 32)).astype(np.float32)
    d1, u1, d2, u2 = (ref.pack(rng.standard_normal(s), BF16) for s in ((16, 64), (32, 16), (3, 64), (32, 3)))
    dx, db, di, out = ctx.to_device(x), ctx.to_device(b), ctx.to_device(np.array([0, 1, 0], dtype=np.int32)), ctx.empty((3, 32))
    need = a.workspace(3)
    space = ctx.empty(need, np.uint8)

    def go():
        a.apply(dx, 3, di, out, base=db, space=space, space_bytes=need)
        return out.numpy()

    assert np.array_equal(go(), b)
    a.load(0, d1, u1, 2.0)
    first = go()
    assert np.array_equal(first[1], b[1]) and not np.array_equal(first[0], b[0])
    a.load(0, d2, u2, 1.0)  # a smaller one: nothing of the larger is left
    want = b[0] + ref.unpack(u2, BF16) @ (ref.unpack(d2, BF16) @ x[0])
    assert np.allclose(go()[0], want, rtol=1e-5, atol=1e-5)
    a.load(0, None, None)
    assert np.array_equal(go(), b)
    a.close()


# ---------------------------------------------------------------------------------------------------------------------------- together
class Graphs:
    """What a caller captures on the ctx stream, through the runtime that the library is linked with."""

    def __init__(self, ctx):
        self.ctx, self.hip = ctx, C.CDLL("libamdhip64.so.7")
        self.stream = C.c_void_p(ctx.L.ps_hip_stream(ctx.h))

    def capture(self, f):
        graph, ready = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # thread local
        f()
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        return lambda: self.hip.hipGraphLaunch(ready, self.stream)


@pytest.mark.parametrize("captured", [False, True])
def test_a_serving_step_together(ctx, hip, captured):
    """Adapters, attention with weights, taking the tokens in, eviction, sampling: twelve steps of four sequences whose caches hold 48 slots, eager and as one captured graph that is replayed, against the
    same steps in 64 bits."""
    rng = np.random.default_rng(11)
    S, H, G, D, n_ctx, keep, width, vocab, steps = 4, 4, 2, 64, 49, 48, 128, 500, 12
    qkv = (H + 2 * G) * D
    a = hip.Adapters(ctx, qkv, width, 3, 8)
    down, up = [ref.pack(rng.standard_normal((8, width)) / 12, BF16) for _ in range(3)], [ref.pack(rng.standard_normal((qkv, 8)) / 3, BF16) for _ in range(3)]
    for i in range(3):
        a.load(i, down[i], up[i], 1.0)
    ids = np.array([0, 2, -1, 0], dtype=np.int32)
    x, base = rng.standard_normal((steps, S, width)).astype(np.float32), rng.standard_normal((steps, S, qkv)).astype(np.float32)
    logits, u = (2 * rng.standard_normal((steps, S, vocab))).astype(np.float32), rng.random((steps, S)).astype(np.float32)
    n_kv = np.array([40, 0, 47, 48], dtype=np.int32)
    k, v = rng.standard_normal((2, S, n_ctx, G, D)).astype(np.float32)
    w = rng.random((S, G, n_ctx)).astype(np.float32)
    pos = np.tile(np.arange(n_ctx, dtype=np.int32), (S, G, 1))
    d = {n: ctx.to_device(y) for n, y in (("x", x[0]), ("base", base[0]), ("logits", logits[0]), ("u", u[0]), ("n", n_kv), ("k", k), ("v", v), ("w", w), ("pos", pos), ("ids", ids),
                                          ("new", n_kv.reshape(S, 1)), ("one", np.ones(S, dtype=np.int32)), ("k_cap", np.full(S, 30, dtype=np.int32)))}
    d["qkv"], d["out"], d["tokens"] = ctx.empty((S, qkv)), ctx.empty((S, H * D)), ctx.empty((S,), np.int32)
    cache = hip.kv_cache(F32, d["k"], d["v"], d["n"], S, n_ctx, G, D, pos=d["pos"], weight=d["w"])
    q = d["qkv"].ptr
    attn = hip.cache_attn_args(q, d["out"], H, 1, 0.125, k_new=q + H * D * 4, v_new=q + (H + G) * D * 4, pos_new=d["new"], weight_out=d["w"], strides=(qkv, qkv, 0, 0, qkv, qkv))
    evict, settings = hip.cache_evict_args(keep, recent=8, first=2), hip.sample_params(u=d["u"], top_k=d["k_cap"])
    need = [ctx.cache_attn_workspace(cache, attn), ctx.cache_evict_workspace(cache, evict), ctx.sample_workspace(vocab, S), a.workspace(S)]
    space = [ctx.empty(max(16, n), np.uint8) for n in need]

    def step():
        a.apply(d["x"], S, d["ids"], d["qkv"], base=d["base"], space=space[3], space_bytes=need[3])
        ctx.cache_attn(cache, attn, space[0], need[0])
        ctx.cache_advance(cache, d["one"])
        ctx.cache_evict(cache, evict, space[1], need[1])
        ctx.sample(d["logits"], vocab, S, settings, d["tokens"], space=space[2], space_bytes=need[2])

    go = Graphs(ctx).capture(step) if captured else step
    K, V, W, P, N = k.astype(np.float64), v.astype(np.float64), w.astype(np.float64), pos.copy(), n_kv.copy()
    for i in range(steps):
        for name, y in (("x", x[i]), ("base", base[i]), ("logits", logits[i]), ("u", u[i]), ("new", (n_kv + i).astype(np.int32).reshape(S, 1))):
            ctx.check(ctx.L.ps_hip_memcpy_h2d(ctx.h, d[name].ptr, np.ascontiguousarray(y).ctypes.data_as(C.c_void_p), y.nbytes))
        go()
        out, tokens, n_now, w_now, p_now = (d[n].numpy() for n in ("out", "tokens", "n", "w", "pos"))
        for s in range(S):
            y = base[i, s].astype(np.float64)
            if ids[s] >= 0:
                y = y + ref.unpack(up[ids[s]], BF16) @ (ref.unpack(down[ids[s]], BF16) @ x[i, s].astype(np.float64))
            K[s, N[s]], V[s, N[s]], P[s, :, N[s]] = y[H * D:(H + G) * D].reshape(G, D), y[(H + G) * D:].reshape(G, D), n_kv[s] + i
            o, ws, _, _ = ref.attend(y[:H * D].reshape(1, H, D), K[s], V[s], int(N[s]), 1, 0.125)
            # differences of earlier steps' fp32 rows and weights stay below 1e-4 of results of order one over these steps: 12 steps of sums of at most 128 + 49 roundings of 2^-24 each, scores up to ~20
            assert np.abs(out[s] - o.reshape(-1)).max() < 1e-4
            W[s, :, :N[s]] += ws[:, :N[s]]
            W[s, :, N[s]] = ws[:, N[s]]
            N[s] += 1
            if N[s] > keep:
                for g in range(G):
                    take = ref.evict(int(N[s]), keep, 8, 2, W[s, g], P[s, g])
                    K[s, :keep, g], V[s, :keep, g], W[s, g, :keep], P[s, g, :keep] = K[s, take, g], V[s, take, g], W[s, g, take], P[s, g, take]
                N[s] = keep
            assert n_now[s] == N[s] and np.array_equal(p_now[s, :, :N[s]], P[s, :, :N[s]])
            assert np.abs(w_now[s, :, :N[s]] - W[s, :, :N[s]]).max() < 1e-4
            assert tokens[s] == ref.sample(logits[i, s], 1.0, 30, 1.0, 0.0, float(u[i, s]))[0]
    a.close()


@pytest.mark.parametrize("dtype,n_new", [(F32, 1), (BF16, 1), (BF16, 24), (F16, 60), (F32, 60)])
def test_captured_steps_are_replayed_with_other_lengths(ctx, hip, dtype, n_new):
    """Two graphs of one step each, with a workspace of their own, replayed in turn over lengths that change in between, eager work between them: the bits of the eager call each time."""
    rng = np.random.default_rng(n_new)
    both = [Step(ctx, hip, rng, dtype, 8, 2, 64, 900, [800, 3, 410], n_new) for _ in range(2)]
    go = [Graphs(ctx).capture(s.run) for s in both]
    for n_kv in ([800, 3, 410], [0, 0, 0], [840, 1, 2], [5, 830, 128]):
        new = np.array(n_kv, dtype=np.int32)
        want = []
        for s in both:
            ctx.check(ctx.L.ps_hip_memcpy_h2d(ctx.h, s.d["n_kv"].ptr, new.ctypes.data_as(C.c_void_p), new.nbytes))
            for n in ("k", "v"):  # (every slot is held by one of the steps: none is to be NaN)
                x = np.nan_to_num(ref.unpack(getattr(s, n), dtype), nan=0.25)
                x = np.ascontiguousarray(ref.pack(x, dtype))
                ctx.check(ctx.L.ps_hip_memcpy_h2d(ctx.h, s.d[n].ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
            s.run()
            want.append([s.d[n].numpy() for n in ("out", "weight_out", "k", "v")])
        for _ in range(2):
            for s in both:  # (results that a replay has to write again)
                x = np.zeros(s.weight.shape, dtype=np.float32)
                ctx.check(ctx.L.ps_hip_memcpy_h2d(ctx.h, s.d["weight_out"].ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
            for g in go:
                assert g() == 0
            ctx.sync()
            for s, w in zip(both, want):
                got = [s.d[n].numpy() for n in ("out", "weight_out", "k", "v")]
                for i, n in enumerate(n_kv):
                    e = n + n_new
                    assert np.array_equal(got[0][i].view(np.uint8), w[0][i].view(np.uint8)) and np.array_equal(got[1][i, :, :e], w[1][i, :, :e])
                assert np.array_equal(got[2].view(np.uint8), w[2].view(np.uint8)) and np.array_equal(got[3].view(np.uint8), w[3].view(np.uint8))
    for s in both:
        s.free()


def test_sampling_eviction_and_adapters_captured_before_any_eager_call(ctx, hip):
    """Captured as the first calls of their kinds in a new context, replayed with other numbers in the same places, sizes that take several kernels each."""
    rng = np.random.default_rng(21)
    mine = hip.Ctx(0)
    rows, n, T, N, K = 3, 50000, 100, 64, 96
    a = hip.Adapters(mine, N, K, 4, 16)
    mats = [(ref.pack(rng.standard_normal((16, K)) / 10, BF16), ref.pack(rng.standard_normal((N, 16)), BF16)) for _ in range(4)]
    for i, (d, u) in enumerate(mats):
        a.load(i, d, u, 1.0)
    up = mine.to_device
    logits, u, ids, prob = up(np.zeros((rows, n), dtype=np.float32)), up(np.zeros(rows, dtype=np.float32)), mine.empty((rows,), np.int32), mine.empty((rows,))
    x, who, out = up(np.zeros((T, K), dtype=np.float32)), up(np.zeros(T, dtype=np.int32)), mine.empty((T, N))
    S, G, n_ctx, D, keep = 2, 2, 600, 8, 200
    k, v, w, pos = (up(y) for y in (np.zeros((S, n_ctx, G, D), np.float32), np.zeros((S, n_ctx, G, D), np.float32), np.zeros((S, G, n_ctx), np.float32), np.zeros((S, G, n_ctx), np.int32)))
    n_kv = up(np.zeros(S, dtype=np.int32))
    cache, evict = hip.kv_cache(F32, k, v, n_kv, S, n_ctx, G, D, pos=pos, weight=w), hip.cache_evict_args(keep, 20, 2)
    need = [mine.sample_workspace(n, rows), a.workspace(T), mine.cache_evict_workspace(cache, evict)]
    space = [mine.empty(b, np.uint8) for b in need]

    def step():
        mine.sample(logits, n, rows, hip.sample_params(u=u), ids, prob=prob, space=space[0], space_bytes=need[0])
        a.apply(x, T, who, out, space=space[1], space_bytes=need[1])
        mine.cache_evict(cache, evict, space[2], need[2])

    go = Graphs(mine).capture(step)

    def put(d, y):
        y = np.ascontiguousarray(y)
        mine.check(mine.L.ps_hip_memcpy_h2d(mine.h, d.ptr, y.ctypes.data_as(C.c_void_p), y.nbytes))
        return y

    for i in range(4):
        l = put(logits, (2 * rng.standard_normal((rows, n))).astype(np.float32))  # noqa: E741
        uu, xx, ww = put(u, rng.random(rows).astype(np.float32)), put(x, rng.standard_normal((T, K)).astype(np.float32)), put(w, rng.random((S, G, n_ctx)).astype(np.float32))
        kk, _, ii = put(k, rng.standard_normal((S, n_ctx, G, D)).astype(np.float32)), put(v, rng.standard_normal((S, n_ctx, G, D)).astype(np.float32)), put(who, rng.integers(-1, 4, T).astype(np.int32))
        pp, nn = put(pos, np.argsort(rng.random((S, G, n_ctx)), -1).astype(np.int32)), put(n_kv, np.array([600, 150 + 40 * i], dtype=np.int32))
        assert go() == 0
        tokens, y, k2, w2 = ids.numpy(), out.numpy(), k.numpy(), w.numpy()
        for r in range(rows):
            want, _, near = ref.sample(l[r], 1.0, 0, 1.0, 0.0, float(uu[r]))
            assert near < 2.0**-25 or tokens[r] == want
        for t in range(T):
            if ii[t] < 0:
                assert (y[t] == 0).all()
                continue
            d, b = (ref.unpack(m, BF16) for m in mats[ii[t]])
            size = np.abs(b) @ (np.abs(d) @ np.abs(xx[t]).astype(np.float64))
            assert (np.abs(y[t] - b @ (d @ xx[t].astype(np.float64))) <= ((K + 3 * 16 + 32) * 2.0**-24 + 2.0**-22) * size).all()
        for s in range(S):
            for g in range(G):
                take = ref.evict(int(nn[s]), keep, 20, 2, ww[s, g], pp[s, g]) if nn[s] > keep else np.arange(nn[s])
                assert np.array_equal(k2[s, :len(take), g], kk[s, take, g]) and np.array_equal(w2[s, g, :len(take)], ww[s, g, take])
        assert np.array_equal(n_kv.numpy(), np.minimum(nn, keep))
    a.close()
