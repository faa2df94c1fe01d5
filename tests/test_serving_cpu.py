"""The entries of a serving step of many sequences on the host, without a GPU (tests/fake_hip.cpp in front of the library): what they refuse, before anything is enqueued, what the workspace functions say, on which
device they launch, and the adapters' memory."""
from test_host_calls import child, fake  # noqa: F401  (fixtures)

MADE = """
ctx = hip.Ctx(0)
a = lambda n=64: ctx.malloc(n)
def cache(dtype=1, S=2, n_ctx=64, G=2, dim=64, pos=True, weight=True, strides=None):
    return hip.kv_cache(dtype, a(), a(), a(), S, n_ctx, G, dim, pos=a() if pos else None, weight=a() if weight else None, strides=strides)
def attn(heads=4, new=3, scale=0.125, **k):
    return hip.cache_attn_args(a(), a(), heads, new, scale, **k)
space = a(1 << 20)
def quiet(f):  # refused, and nothing enqueued
    fake.fake_reset()
    why = refused(f)
    assert count("hipLaunchKernel") == count("hipMemcpy") == count("hipMemset") == 0, why
    return why
"""


def test_attention_refuses_what_it_cannot_do(child):  # noqa: F811
    child(MADE + """
def go(c, p, ws=space, n=1 << 20): return quiet(lambda: ctx.cache_attn(c, p, ws, n))
assert "type" in go(cache(dtype=8), attn())
for dim in (0, 4, 12, 136, 256): assert "size" in go(cache(dim=dim), attn())
for n_ctx in (0, -1, (1 << 28) + 1): go(cache(n_ctx=n_ctx), attn())
assert "slots" in go(cache(G=0), attn())
assert "many" in go(cache(S=65536), attn())
assert "aligned" in go(cache(strides=(8192, 132, 64)), attn()) and "aligned" in go(cache(strides=(8192, 128, 4)), attn()) and "aligned" in go(cache(strides=(8190, 128, 64)), attn())
for heads in (0, 3, -2): assert "query heads" in go(cache(), attn(heads=heads))
for new in (-1, 65): assert "new tokens" in go(cache(), attn(new=new))
for scale in (float("nan"), float("inf"), 2e30): assert "scale" in go(cache(), attn(scale=scale))
c = cache(); c.k = None
assert "missing" in go(c, attn())
c = cache(); c.v = c.k
assert "same" in go(c, attn())
c = cache(); c.n_kv = None
assert "missing" in go(c, attn())
c = cache(); c.k += 8
assert "aligned" in go(c, attn())
p = attn(); p.out = p.q
assert "same" in go(cache(), p)
p = attn(); p.q = None
assert "missing" in go(cache(), p)
assert "together" in go(cache(), attn(k_new=a())) and "together" in go(cache(), attn(v_new=a()))
assert "positions" in go(cache(pos=False), attn(pos_new=a()))
assert "new keys" in go(cache(), attn(pos_new=a()))
for i in range(6):
    assert "aligned" in go(cache(), attn(strides=[4 if i == j else 0 for j in range(6)])), i
p = attn(); p.q += 4
assert "aligned" in go(cache(), p)
need = ctx.cache_attn_workspace(cache(), attn())
assert need > 0
for ws, n in ((None, need), (space, need - 1), (space + 8, need), (space, 0)): assert "workspace" in go(cache(), attn(), ws, n)
assert "many" in go(cache(S=60000, n_ctx=1 << 27), attn(new=1 << 20))
assert "many" in go(cache(dtype=0, S=65535, G=8, n_ctx=4096, dim=8), attn(heads=8, new=100, weight_out=a()))  # 64 slots a work-group: more than 2^24 of them
assert "many" in go(cache(S=65535, G=512, n_ctx=16, dim=8), attn(heads=512, new=1))
c, p = cache(dtype=0, S=500, G=512, n_ctx=4096, dim=8), attn(heads=512, new=512)  # 8 parts of 512 slots, 16 work-groups of 32 rows each: a grid of more than 2^32 threads; there are 4
heads, row_tiles, part = 500 * 512, 512 // 16, 16 * (8 + 2) * 4
assert ctx.cache_attn_workspace(c, p) == heads * 512 * 4 + heads * row_tiles * 4 * part
fake.fake_reset()
ctx.cache_attn(cache(), attn(), space, need)
assert count("hipLaunchKernel") > 0
# nothing to do is no error
fake.fake_reset()
ctx.cache_attn(cache(), attn(new=0), None, 0)
ctx.cache_attn(cache(S=0), attn(), None, 0)
assert count("hipLaunchKernel") == 0 and ctx.cache_attn_workspace(cache(), attn(new=0)) == ctx.cache_attn_workspace(cache(dim=12), attn()) == 0
quiet(lambda: ctx.cache_advance(cache(), None))
quiet(lambda: ctx.cache_advance(cache(), a(), a(), -1))
""")


def test_eviction_refuses_what_it_cannot_do(child):  # noqa: F811
    child(MADE + """
def go(c, p, ws=space, n=1 << 20): return quiet(lambda: ctx.cache_evict(c, p, ws, n))
for keep, recent, first in ((0, 0, 0), (-1, 0, 0), (5, 6, 0), (5, 3, 3), (5, -1, 0), (5, 0, -1), (2**31 - 1, 2**31 - 1, 2**31 - 1)):
    assert "keep" in go(cache(), hip.cache_evict_args(keep, recent, first))
assert "positions" in go(cache(pos=False), hip.cache_evict_args(8)) and "positions" in go(cache(weight=False), hip.cache_evict_args(8))
assert "type" in go(cache(dtype=26), hip.cache_evict_args(8))
need = ctx.cache_evict_workspace(cache(), hip.cache_evict_args(8))
for ws, n in ((None, need), (space, need - 1), (space + 8, need)): assert "workspace" in go(cache(), hip.cache_evict_args(8), ws, n)
fake.fake_reset()
ctx.cache_evict(cache(), hip.cache_evict_args(8), space, need)
ctx.cache_evict(cache(), hip.cache_evict_args(100), space, need)  # more than there are slots
assert count("hipLaunchKernel") == 4
ctx.cache_evict(cache(S=0), hip.cache_evict_args(8), None, 0)
assert count("hipLaunchKernel") == 4
""")


def test_sampling_refuses_what_it_cannot_do(child):  # noqa: F811
    child(MADE + """
u = hip.sample_params(a())
def go(n=1000, rows=2, p=u, logits=a(), ids=a(), dtype=0, stride=None, ws=space, b=1 << 20): return quiet(lambda: ctx.sample(logits, n, rows, p, ids, dtype=dtype, stride=stride, space=ws, space_bytes=b))
for n in (0, -5, (1 << 24) + 1): assert "logits" in go(n=n)
assert "rows" in go(rows=-1) and "rows" in go(rows=1 << 31)
assert "rows" in go(n=10, rows=1 << 22)  # 1024 threads each: a grid would pass 2^32 of them
for dtype in (2, 26, 99): assert "F32" in go(dtype=dtype)
assert "overlap" in go(stride=999)
assert "random" in go(p=hip.sample_params(None))
assert "missing" in go(logits=None) and "missing" in go(ids=None) and "aligned" in go(logits=a() + 2)
need = ctx.sample_workspace(100000, 2)
assert need > 0 and "workspace" in go(n=100000, b=need - 1) and "workspace" in go(n=100000, ws=None) and "workspace" in go(n=100000, ws=space + 4)
assert ctx.sample_workspace(1000, 500) == 0 and ctx.sample_workspace(0, 1) == 0 and ctx.sample_workspace(5, 0) == 0
fake.fake_reset()
ctx.sample(a(), 1000, 500, u, a())  # rows enough that each has a work-group: no workspace
assert count("hipLaunchKernel") == 1
ctx.sample(None, 1000, 0, u, None)
assert count("hipLaunchKernel") == 1
""")


def test_adapters_refuse_what_they_cannot_do(child):  # noqa: F811
    child(MADE + """
for N, K, slots, rank in ((0, 8, 1, 1), (8, 0, 1, 1), (8, 8, 0, 1), (8, 8, 1, 0), (8, 8, 1, 257), (8, 8, 65537, 1), ((1 << 24) + 1, 8, 1, 1), (8, 8, -1, 1)):
    quiet(lambda: hip.Adapters(ctx, N, K, slots, rank))
s = hip.Adapters(ctx, 8, 12, 2, 4)
down, up = np.ones((3, 12), dtype=np.uint16), np.ones((8, 3), dtype=np.uint16)
s.load(1, down, up, 2.0)
s.load(1, None, None)
for slot in (-1, 2): assert "slot" in quiet(lambda: s.load(slot, down, up))
for d, u in ((down[:, :11], up), (down, up[:7]), (down, up[:, :2]), (down.astype(np.float32), up), (np.ones((5, 12), dtype=np.uint16), np.ones((8, 5), dtype=np.uint16))): quiet(lambda: s.load(0, d, u))
assert "matrices" in quiet(lambda: ctx.check(ctx.L.ps_hip_adapters_load(ctx.h, s.h, 0, None, None, 2, 1.0)))
need = s.workspace(5)
def go(x=a(), T=5, ids=a(), out=a(), ws=space, n=need, **k): return quiet(lambda: s.apply(x, T, ids, out, space=ws, space_bytes=n, **k))
assert "x must be" in go(dtype=1)
assert "tokens" in go(T=-1) and "tokens" in go(T=(1 << 22) + 1)
for k in ({"x": None}, {"ids": None}, {"out": None}, {"x": a() + 2}): assert "missing" in go(**k)
x = a()
assert "same" in go(x=x, out=x)
assert "overlap" in go(ldx=11) and "overlap" in go(ldo=7)
for ws, n in ((None, need), (space, need - 1), (space + 8, need)): assert "workspace" in go(ws=ws, n=n)
fake.fake_reset()
s.apply(a(), 0, a(), a())
assert count("hipLaunchKernel") == 0 and s.workspace(0) == 0
other = hip.Ctx(1)
assert "device" in refused(lambda: other.check(other.L.ps_hip_adapters_apply(other.h, s.h, 0, a(), 12, 5, a(), None, a(), 8, space, 1 << 20)))
s.close()
s.close()
""")


def test_adapters_give_their_memory_back(child):  # noqa: F811
    """closed, and where the n-th allocation or copy of a set fails"""
    child(MADE + """
held = fake.fake_held()
s = hip.Adapters(ctx, 80, 120, 5, 20)
s.load(4, np.ones((17, 120), dtype=np.uint16), np.ones((80, 17), dtype=np.uint16), 2.0)
assert fake.fake_held() > held and fake.fake_stray() == 0
s.close()
assert fake.fake_held() == held
for n in (1, 2, 3, 4):
    fail("hipMalloc", n)
    refused(lambda: hip.Adapters(ctx, 80, 120, 5, 20))
    assert fake.fake_held() == held, n
s = hip.Adapters(ctx, 80, 120, 5, 20)
fail("hipMemcpyAsync", 2)
refused(lambda: s.load(0, np.ones((17, 120), dtype=np.uint16), np.ones((80, 17), dtype=np.uint16)))
s.load(0, np.ones((17, 120), dtype=np.uint16), np.ones((80, 17), dtype=np.uint16))
s.close()
assert fake.fake_held() == held
""")


def test_launches_go_to_the_contexts_device_and_leave_the_callers_current(child):  # noqa: F811
    child(MADE + """
dev = C.c_int()
other = hip.Ctx(1)  # (its device is current now)
def current():
    fake.hipGetDevice(C.byref(dev))
    return dev.value
assert current() == 1
c, p, x, y, s = cache(), attn(), a(), a(), hip.sample_params(a())
calls = [lambda: ctx.cache_attn(c, p, space, 1 << 20), lambda: ctx.cache_advance(c, x), lambda: ctx.cache_evict(c, hip.cache_evict_args(8), space, 1 << 20), lambda: ctx.sample(x, 100, 300, s, y)]
for f in calls:
    fake.hipSetDevice(1)
    fake.fake_reset()
    f()
    assert count("hipLaunchKernel") >= 1 and current() == 1
# what a failing launch says is the caller's to see
fail("hipLaunchKernel")
try: ctx.sample(x, 100, 300, s, y)
except hip.PSHipError: pass
else: raise AssertionError("a failed launch went unnoticed")
""")


def test_everything_of_a_step_is_captured(child):  # noqa: F811
    """nothing but launches between the beginning and the end of a capture: no allocation, no copy, no memset, no wait"""
    child(MADE + """
s = hip.Adapters(ctx, 8, 12, 2, 4)
fake.fake_reset()
ctx.cache_attn(cache(), attn(weight_out=a(), tree=a()), space, 1 << 20)
ctx.cache_attn(cache(dtype=30), attn(new=40, weight_out=a()), space, 1 << 20)
ctx.cache_advance(cache(), a(), a(), 3)
ctx.cache_evict(cache(), hip.cache_evict_args(8), space, 1 << 20)
ctx.sample(a(), 100000, 2, hip.sample_params(a()), a(), space=space, space_bytes=1 << 20) if ctx.sample_workspace(100000, 2) <= 1 << 20 else None
s.apply(a(), 500, a(), a(), space=space, space_bytes=1 << 20)
assert count("hipLaunchKernel") > 10 and count("hipMemcpy") == count("hipMemset") == count("Synchronize") == count("hipEvent") == 0
# (the lambdas allocate their buffers through the library: no other allocation)
""")


def test_a_workspace_serves_every_smaller_call(child):  # noqa: F811
    """what the workspace functions say is enough for fewer sequences, new tokens, rows or tokens too: a server keeps one for its largest step"""
    child(MADE + """
import random
rng = random.Random(1)
huge = C.c_void_p(a())  # (nothing is enqueued for real: an address that is aligned will do)
for n, rows in ((128256, 256), (128256, 129), (128256, 128), (151936, 33), (4096, 128), (50000, 7), (8192, 100)):
    have = ctx.sample_workspace(n, rows)
    for r in sorted({1, 2, 3, rows, *(rng.randint(1, rows) for _ in range(30)), *(x for x in (16, 31, 32, 33, 63, 64, 65, 127, 128) if x <= rows)}):
        for m in (n, n // 2, n // 3, 5000, 4096, 100):
            for dtype in (0, 1, 30):
                if m <= n: ctx.sample(a(), m, r, hip.sample_params(a()), a(), dtype=dtype, space=huge.value, space_bytes=have)
for N, K, slots, rank in ((64, 4096, 8, 64), (14336, 4096, 64, 64), (2048, 2048, 3, 16), (1 << 20, 300, 100, 4), (128, 64, 9000, 2)):
    s = hip.Adapters(ctx, N, K, slots, rank)
    for T in (1, 127, 128, 253, 300, 5000):
        have = s.workspace(T)
        for t in range(1, T + 1, 1 if T < 400 else 37): s.apply(a(), t, a(), a(), space=huge.value, space_bytes=have)
    s.close()
for i in range(400):
    dtype, S, G, dim = rng.choice((0, 1, 30)), rng.choice((1, 2, 4, 16, 32, 255, 256, 257, 300, 600)), rng.choice((1, 2, 8)), rng.choice((8, 64, 128))
    heads, n_ctx, new = G * rng.choice((1, 4, 7, 33, 150)), rng.choice((100, 129, 300, 600, 1100, 4096, 8192, 100000)), rng.choice((1, 2, 8, 9, 24, 33, 64, 70, 100))
    weights = {"weight_out": a()} if rng.random() < 0.6 else {}
    have = ctx.cache_attn_workspace(cache(dtype, S, n_ctx, G, dim), attn(heads, new, **weights))
    assert have
    for s in {1, min(2, S), S, *(rng.randint(1, S) for _ in range(8)), *(x for x in (255, 256, 257) if x < S)}:
        for t in {1, new, *(rng.randint(1, new) for _ in range(8)), *(x for x in (4, 5, 8, 9, 16, 17, 32, 33) if x < new)}:
            for w in {0, len(weights)}:
                ctx.cache_attn(cache(dtype, s, n_ctx, G, dim), attn(heads, t, **(weights if w else {})), huge.value, have)
    e = hip.cache_evict_args(rng.choice((1, 50, 99)))
    have = ctx.cache_evict_workspace(cache(dtype, S, n_ctx, G, dim), e)
    for s in {1, S, rng.randint(1, S)}: ctx.cache_evict(cache(dtype, s, n_ctx, G, dim), e, huge.value, have)
""")


def test_adapters_with_infinite_numbers_are_refused(child):  # noqa: F811
    """in either matrix, of either sign, in the last place too; the slot keeps what it had, the largest number and NaN are taken"""
    child(MADE + """
s = hip.Adapters(ctx, 8, 12, 2, 4)
ones = lambda *shape: np.full(shape, 0x3f80, dtype=np.uint16)
s.load(1, ones(3, 12), ones(8, 3))
for bits in (0x7f80, 0xff80):
    for i, j in ((0, 0), (2, 11), (1, 5)):
        down = ones(3, 12)
        down[i, j] = bits
        assert "infinite" in quiet(lambda: s.load(1, down, ones(8, 3)))
    for i, j in ((0, 0), (7, 2)):
        up = ones(8, 3)
        up[i, j] = bits
        assert "infinite" in quiet(lambda: s.load(1, ones(3, 12), up))
for bits in (0x7f7f, 0xff7f, 0x7fc0, 0x7f81, 0x0001):
    s.load(1, np.full((3, 12), bits, dtype=np.uint16), np.full((8, 3), bits, dtype=np.uint16))
""")


def test_each_operator_of_a_step_is_its_launches_and_nothing_else(child):  # noqa: F811
    """every operator, the sampler in parts among them, alone between two looks at the counts: so many launches, and no allocation, copy, memset, wait or event"""
    child(MADE + """
s = hip.Adapters(ctx, 8, 12, 2, 4)
s.load(0, np.ones((3, 12), dtype=np.uint16), np.ones((8, 3), dtype=np.uint16))
c, c16, tree = cache(), cache(dtype=30), a()
one, two, many = attn(weight_out=a(), tree=tree), attn(new=3), attn(new=40, k_new=a(), v_new=a(), weight_out=a())
long_one = cache(dtype=30, S=3, n_ctx=4096)
evict, settings, x, y, z, e = hip.cache_evict_args(8), hip.sample_params(a()), a(), a(), a(), a()
room = max(ctx.sample_workspace(100000, 2), ctx.cache_attn_workspace(long_one, many), s.workspace(500), 1 << 20)
ws = a(room)
for launches, call in (
    (2, lambda: ctx.cache_attn(c, one, ws, room)),           # rows in one part, weights from the scores
    (1, lambda: ctx.cache_attn(c, two, ws, room)),
    (2, lambda: ctx.cache_attn(long_one, two, ws, room)),    # parts and their join
    (5, lambda: ctx.cache_attn(long_one, many, ws, room)),   # new rows, rows, join, weights, their sums
    (4, lambda: ctx.cache_attn(c16, many, ws, room)),        # one part
    (1, lambda: ctx.cache_advance(c, x)), (2, lambda: ctx.cache_advance(c, x, y, 3)),
    (2, lambda: ctx.cache_evict(c, evict, ws, room)),
    (3, lambda: ctx.sample(x, 100000, 2, settings, y, prob=z, space=ws, space_bytes=room)), (1, lambda: ctx.sample(x, 100000, 200, settings, y, space=ws, space_bytes=room)),
    (2, lambda: s.apply(x, 5, y, z, base=e, space=ws, space_bytes=room)), (3, lambda: s.apply(x, 500, y, z, space=ws, space_bytes=room)),
):
    fake.fake_reset()
    call()
    assert count("hipLaunchKernel") == launches, (launches, count("hipLaunchKernel"))
    for name in ("hipMalloc", "hipHostMalloc", "hipFree", "hipMemcpyAsync", "hipMemsetAsync", "hipStreamSynchronize", "hipDeviceSynchronize", "hipEventRecord", "hipEventSynchronize", "put_kernel", "pin_copy_kernel"):
        assert count(name) == 0, (launches, name)
""")


def test_adapters_launch_on_the_contexts_device_and_leave_the_callers_current(child):  # noqa: F811
    child(MADE + """
dev = C.c_int()
s = hip.Adapters(ctx, 8, 12, 2, 4)
other = hip.Ctx(1)
def current():
    fake.hipGetDevice(C.byref(dev))
    return dev.value
x, y, z = a(), a(), a()
for f in (lambda: s.apply(x, 5, y, z, space=space, space_bytes=1 << 20), lambda: s.load(0, np.ones((3, 12), dtype=np.uint16), np.ones((8, 3), dtype=np.uint16)), lambda: hip.Adapters(ctx, 8, 12, 2, 4)):
    for d in (1, 0):
        fake.hipSetDevice(d)
        fake.fake_reset()
        f()
        assert current() == d and count("hipSetDevice") == 2 * d, (d, count("hipSetDevice"))
""")


def test_arrays_that_are_not_the_devices_or_not_of_the_type_are_refused(child):  # noqa: F811
    """host tensors and numpy arrays, freed arrays, 64-bit lengths, views with gaps: refused where the address is taken, not read on the device"""
    child(MADE + """
import torch
class On:  # a tensor as one on the device looks
    def __init__(self, x): self.x, self.dtype, self.shape, self.device = x, x.dtype, x.shape, torch.device("cuda", 0)
    def data_ptr(self): return self.x.data_ptr()
    def is_contiguous(self): return self.x.is_contiguous()
dev = lambda *s, dtype=torch.int32: On(torch.zeros(*s, dtype=dtype))
k = a()
def made(n_kv, **more): return lambda: hip.kv_cache(0, k, k + 64, n_kv, 2, 64, 2, 64, **more)
freed = ctx.to_device(np.zeros(2, np.int32))
made(freed)()
made(dev(2))()
assert "host" in refused(made(torch.zeros(2, dtype=torch.int32))) and "device memory" in refused(made(np.zeros(2, np.int32))) and "device memory" in refused(made([0, 0]))
assert "int32" in refused(made(dev(2, dtype=torch.int64))) and "int32" in refused(made(dev(2, dtype=torch.float32))) and "int32" in refused(made(ctx.to_device(np.zeros(2, np.int64))))
assert "behind the other" in refused(made(On(torch.zeros(1, dtype=torch.int32).expand(2)))) and "behind the other" in refused(made(On(torch.zeros(4, dtype=torch.int32)[::2])))
freed.free()
assert "freed" in refused(made(freed))
assert "float32" in refused(made(dev(2), weight=dev(2, 2, 64, dtype=torch.float64))) and "int32" in refused(made(dev(2), pos=dev(2, 2, 64, dtype=torch.int64)))
made(dev(2), weight=dev(2, 2, 64, dtype=torch.float32), pos=dev(2, 2, 64))()
made(ctx.to_device(np.zeros(8, np.uint8)))()  # a piece of somebody's memory
q = On(torch.zeros(2, 3, 4, 64))
hip.cache_attn_args(q, k, 4, 3, 0.1, tree=dev(2, 3, 3, dtype=torch.bool), count=dev(2))
hip.cache_attn_args(q, k, 4, 3, 0.1, tree=dev(2, 3, 3, dtype=torch.uint8))
for x in ({"tree": dev(2, 3, 3)}, {"count": dev(2, dtype=torch.int64)}, {"weight_out": dev(2)}, {"pos_new": dev(2, 3, dtype=torch.int64)}, {"k_new": torch.zeros(4)}):
    refused(lambda: hip.cache_attn_args(q, k, 4, 3, 0.1, **x))
for x in ({"u": dev(2, dtype=torch.float64)}, {"u": k, "top_k": dev(2, dtype=torch.int64)}, {"u": k, "temperature": torch.ones(2)}, {"u": k, "min_p": On(torch.zeros(1).expand(2))}): refused(lambda: hip.sample_params(**x))
refused(lambda: hip.cache_evict_args(5, n_kv_out=dev(2, dtype=torch.int64)))
p = hip.sample_params(k)
fake.fake_reset()
refused(lambda: ctx.sample(np.zeros((2, 9), np.float32), 9, 2, p, k))
refused(lambda: ctx.sample(k, 9, 2, p, dev(2, dtype=torch.int64)))
refused(lambda: ctx.cache_advance(cache(), dev(2, dtype=torch.int64)))
s = hip.Adapters(ctx, 8, 12, 2, 4)
refused(lambda: s.apply(k, 5, dev(5, dtype=torch.int64), k, space=space, space_bytes=1 << 20))
assert count("hipLaunchKernel") == 0
""")


def test_arrays_of_other_numbers_than_the_call_says_are_refused(child):  # noqa: F811
    """16-bit logits read as fp32 would be read past their end: an array that knows its type has to have the call's"""
    child(MADE + """
import torch
class On:
    def __init__(self, *s, dtype): self.x = torch.zeros(*s, dtype=dtype); self.dtype, self.shape = dtype, self.x.shape
    def data_ptr(self): return (self.x.data_ptr() + 15) // 16 * 16
    def is_contiguous(self): return True
f32, f16, b16 = torch.float32, torch.float16, torch.bfloat16
u, ids = a(), a()
p = hip.sample_params(u)
fake.fake_reset()
for dtype, good, bad in ((hip.F32, (f32,), (f16, b16, torch.float64, torch.int16)), (hip.F16, (f16, torch.int16), (f32, b16)), (hip.BF16, (b16, torch.int16, torch.uint8), (f32, f16, torch.float64))):
    for t in bad:
        x = On(999, dtype=t)
        for f in (lambda: ctx.sample(x, 100, 3, p, ids, dtype=dtype), lambda: hip.kv_cache(dtype, x, u, u, 2, 64, 2, 64), lambda: hip.kv_cache(dtype, u, x, u, 2, 64, 2, 64)): assert "type" in refused(f)
    for t in good:
        x = On(999, dtype=t)
        ctx.sample(x, 100, 3, p, ids, dtype=dtype)
        hip.kv_cache(dtype, x, u, u, 2, 64, 2, 64)
assert count("hipLaunchKernel") == 6
s = hip.Adapters(ctx, 8, 12, 2, 4)
for x, dtype, base, out in ((On(60, dtype=b16), hip.F32, None, u), (On(60, dtype=f32), hip.BF16, None, u), (On(60, dtype=f32), hip.F32, On(40, dtype=b16), u), (On(60, dtype=f32), hip.F32, None, On(40, dtype=f16))):
    assert "type" in quiet(lambda: s.apply(x, 5, ids, out, base=base, dtype=dtype, space=space, space_bytes=1 << 20))
s.apply(On(60, dtype=b16), 5, ids, On(40, dtype=f32), dtype=hip.BF16, space=space, space_bytes=1 << 20)
for dtype, good, bad in ((hip.F32, f32, b16), (hip.BF16, b16, f32), (hip.F16, f16, b16)):
    c = cache(dtype=dtype)
    for i in range(4):
        for t in (good, bad):
            x = [On(2, 3, 4, 64, dtype=t if i == j else good) for j in range(4)]
            q = hip.cache_attn_args(x[0], x[1], 4, 3, 0.1, k_new=x[2], v_new=x[3])
            if t is good: ctx.cache_attn(c, q, space, 1 << 20)
            else: assert "type" in quiet(lambda: ctx.cache_attn(c, q, space, 1 << 20))
""")


def test_views_whose_rows_have_strides_come_with_them(child):  # noqa: F811
    child(MADE + """
import torch
class On:
    def __init__(self, x): self.x, self.dtype, self.shape = x, x.dtype, x.shape
    def data_ptr(self): return (self.x.data_ptr() + 15) // 16 * 16
    def is_contiguous(self): return self.x.is_contiguous()
u, ids = a(), a()
p = hip.sample_params(u)
part = lambda *s: On(torch.zeros(*s, dtype=torch.float32)[..., :8])  # the first columns of wider rows
s = hip.Adapters(ctx, 8, 8, 2, 4)
w = {"space": space, "space_bytes": 1 << 20}
wide = part(2, 3, 4, 64)
for view, told in (
    (lambda: hip.kv_cache(0, wide, u, u, 2, 3, 4, 8), lambda: hip.kv_cache(0, wide, u, u, 2, 3, 4, 8, strides=(768, 256, 64))),
    (lambda: hip.kv_cache(0, u, wide, u, 2, 3, 4, 8), lambda: hip.kv_cache(0, u, wide, u, 2, 3, 4, 8, strides=(768, 256, 64))),
    (lambda: hip.cache_attn_args(wide, u, 1, 3, 0.1), lambda: hip.cache_attn_args(wide, u, 1, 3, 0.1, strides=(192, 64, 0, 0, 0, 0))),
    (lambda: hip.cache_attn_args(u, wide, 1, 3, 0.1), lambda: hip.cache_attn_args(u, wide, 1, 3, 0.1, strides=(0, 0, 192, 64, 0, 0))),
    (lambda: hip.cache_attn_args(u, u, 1, 3, 0.1, k_new=wide), lambda: hip.cache_attn_args(u, u, 1, 3, 0.1, k_new=wide, v_new=wide, strides=(0, 0, 0, 0, 192, 64))),
    (lambda: hip.cache_attn_args(u, u, 1, 3, 0.1, v_new=wide), lambda: None),
    (lambda: ctx.sample(part(3, 20), 8, 3, p, ids), lambda: ctx.sample(part(3, 20), 8, 3, p, ids, stride=20)),
    (lambda: s.apply(part(3, 20), 3, ids, u, **w), lambda: s.apply(part(3, 20), 3, ids, u, ldx=20, **w)),
    (lambda: s.apply(u, 3, ids, part(3, 20), **w), lambda: s.apply(u, 3, ids, part(3, 20), ldo=20, **w)),
    (lambda: s.apply(u, 3, ids, ids, base=part(3, 20), **w), lambda: s.apply(u, 3, ids, ids, base=part(3, 20), ldo=20, **w)),
):
    assert "without strides" in quiet(view)
    told()
""")
