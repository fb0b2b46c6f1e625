"""The KV cache in blocks on the GPU: tables, append, read-back and attention against paged_ref, alone and in a run."""
import numpy as np
import pytest

import llaisys_amd as L
import paged_ref as ref
from llaisys_amd.hostfmt import f32_to_bf16

pytestmark = pytest.mark.gpu

AMD = dict(device=L.DeviceType.AMD, device_id=0)
DT = {"f32": L.DataType.F32, "bf16": L.DataType.BF16, "f16": L.DataType.F16}
# a weight of the softmax enters the values' product in f16: rounded once for bf16 rows, in two parts for the others
WEIGHT_STEP = {"f32": 2.0 ** -21, "bf16": 2.0 ** -11, "f16": 2.0 ** -21}


def dev(a, dt=None):
    return L.Tensor.from_numpy(np.ascontiguousarray(a), dt, **AMD)


def host(x, dt):
    return f32_to_bf16(x.astype(np.float32)) if dt == "bf16" else x.astype({"f32": np.float32, "f16": np.float16}[dt])


# ---- tables ----------------------------------------------------------------------------------


class Tables:
    """A step's tensors on the GPU and its reference."""

    def __init__(self, old, new, block, rows, width=None, ring=None, head=0, spare=4, seed=0):
        rng = np.random.default_rng(seed)
        nb = lambda n: -(-n // block)
        self.old, self.new, self.block, self.rows = np.array(old, np.int32), np.array(new, np.int32), block, rows
        need = sum(max(0, nb(n) - nb(o)) for o, n in zip(old, new))
        held = sum(max(0, nb(o)) for o in old)
        width = width or max(1, *(max(nb(o), nb(n)) for o, n in zip(old, new))) + 1
        ids = rng.permutation(held + need + spare).astype(np.int32)
        self.table = np.full((len(old), width), -7, np.int32)
        at = 0
        for r, o in enumerate(old):
            k = max(0, nb(o))
            self.table[r, :k] = ids[at:at + k]
            at += k
        free = need + spare if ring is None else ring
        self.ring = np.full(held + need + spare, -9, np.int32)
        self.ring[(head + np.arange(free)) % len(self.ring)] = ids[at:at + free]
        self.state = np.array([head, head + free], np.int64)

    def run(self, in_place=False):
        t, ring, state = dev(self.table), dev(self.ring), dev(self.state)
        out = state if in_place else L.Tensor((2,), L.DataType.I64, **AMD)
        slots, pos = dev(np.full(self.rows, 77, np.int64)), dev(np.full(self.rows, 77, np.int64))
        starts = dev(np.full(len(self.old) + 1, 77, np.int32))
        L.Ops.paged_tables(t, slots, pos, starts, out, dev(self.old), dev(self.new), ring, state, self.block)
        err = L.take_device_error()
        return err, [x.numpy() for x in (t, ring, out, slots, pos, starts)]

    def check(self, in_place=False):
        err, got = self.run(in_place)
        exp = ref.tables(self.table, self.ring, self.state, self.old, self.new, self.block, self.rows)
        assert exp is not None and err == 0
        for name, g, e in zip(("table", "ring", "state", "slots", "pos", "starts"), got, exp):
            assert np.array_equal(g, e), name

    def refused(self):
        err, (t, ring, out, slots, pos, starts) = self.run()
        assert ref.tables(self.table, self.ring, self.state, self.old, self.new, self.block, self.rows) is None
        assert err == 2
        assert np.array_equal(t, self.table) and np.array_equal(ring, self.ring) and np.array_equal(out, self.state)
        assert (slots == -1).all() and (pos == 0).all() and (starts == 0).all()


def _lens(n, most, seed):
    rng = np.random.default_rng(seed)
    return [int(x) for x in np.exp(rng.uniform(0, np.log(most + 1), n)) - 1]


@pytest.mark.parametrize("block", [16, 64, 256])
@pytest.mark.parametrize("requests,most", [(1, 1), (1, 5000), (3, 40), (64, 300), (65, 900), (1100, 200), (2500, 40)])
def test_tables(block, requests, most):
    old, new = _lens(requests, most, 1), _lens(requests, most, 2)
    rows = sum(max(0, n - o) for o, n in zip(old, new))
    Tables(old, new, block, rows + 5, head=123).check()
    Tables(old, [o + 1 for o in old], block, requests, head=3).check(in_place=True)


def test_tables_edges():
    Tables([0], [0], 16, 0).check()  # nothing to do, no rows
    Tables([0, 16, 32], [16, 16, 33], 16, 17).check()  # exact ends of blocks
    Tables([33, 0, 5], [0, 48, 5], 16, 48, ring=0, spare=0).check(in_place=True)  # blocks given back are taken in the same step
    Tables([100, 7, 64], [0, 0, 0], 16, 3, ring=2).check()  # all end
    Tables([0], [70000], 16, 70000, head=10 ** 12).check()  # one long prompt, a ring that has turned many times
    # many groups of threads, a state updated in place, blocks given back and taken in the same step
    Tables([12000, 5, 0, 700, 64], [0, 4000, 8000, 1, 70], 16, 13000, head=77, ring=0, spare=0).check(in_place=True)
    Tables([9000, 5, 0, 700, 64], [0, 4000, 8000, 1, 70], 16, 13000, head=77, spare=9).check()
    Tables(_lens(8192, 30, 5), _lens(8192, 60, 6), 16, 200000, head=5).check(in_place=True)


def test_tables_refuse_what_cannot_be_done():
    Tables([0, 5], [40, 9], 16, 43).refused()  # one row too few
    Tables([0], [100], 16, 100, ring=6).refused()  # one block too few
    Tables([0], [100], 16, 100, width=6).refused()  # the table is too narrow
    Tables([0, -1], [10, 10], 16, 30).refused()
    Tables([4, 1], [10, -10], 16, 30).refused()
    t = Tables([40], [0], 16, 1)
    t.state[1] = t.state[0] + len(t.ring) - 1  # giving back would run over the head
    t.refused()
    t = Tables([0], [10], 16, 10)
    t.state[:] = t.state[::-1]
    t.refused()


# ---- append and read-back --------------------------------------------------------------------


class Cache:
    def __init__(self, n_blocks, heads, block, dim, seed=0):
        rng = np.random.default_rng(seed)
        shape = (n_blocks, heads, block, dim)
        self.k, self.v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (rng.uniform(0.01, 0.03, shape[:2]).astype(np.float32) for _ in range(2))

    def tensors(self):
        return [dev(self.k), dev(self.ks), dev(self.v), dev(self.vs)]


def _slots(lens, block, n_blocks, pad=0, seed=0):
    """Slots of requests that go from lens[i][0] to lens[i][1] tokens, in blocks of any order."""
    ids, at, out = np.random.default_rng(seed).permutation(n_blocks), 0, []
    for o, n in lens:
        p = np.arange(o, n)
        out.append(ids[at + p // block] * block + p % block)
        at += -(-n // block)
    assert at <= n_blocks
    return np.concatenate(out + [np.full(pad, -1)]).astype(np.int64)


def _check_append(cache, k, v, slots, dt):
    t = cache.tensors()
    L.Ops.paged_kv_append_int8(*t, dev(k, DT[dt]), dev(v, DT[dt]), dev(slots))
    assert L.take_device_error() == 0
    for codes, scales, x, (c0, s0) in ((t[0], t[1], k, (cache.k, cache.ks)), (t[2], t[3], v, (cache.v, cache.vs))):
        ec, es = ref.append(c0, s0, x, slots)
        assert np.array_equal(scales.numpy().view(np.uint32), es.view(np.uint32))
        assert np.array_equal(codes.numpy(), ec)
    return t


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,dim,block", [(2, 128, 64), (1, 16, 16), (3, 80, 16), (2, 64, 256), (1, 256, 32)])
def test_append_and_read(dt, heads, dim, block):
    rng = np.random.default_rng(dim + block)
    lens = [(0, 1), (block - 1, block + 1), (3, 3 * block + 5), (0, block), (block, 2 * block), (7, 8), (5, 300)]
    n_blocks = sum(-(-n // block) for _, n in lens) + 2
    slots = _slots(lens, block, n_blocks, pad=3)
    k, v = (host(rng.standard_normal((len(slots), heads, dim)) * rng.choice([0.1, 1, 4], (len(slots), 1, 1)), dt) for _ in range(2))
    cache = Cache(n_blocks, heads, block, dim)
    t = _check_append(cache, k, v, slots, dt)
    ask = np.concatenate([rng.permutation(n_blocks * block)[:517], [-1]])
    back = [dev(np.full((len(ask), heads, dim), 0x4242, np.uint16) if dt == "bf16" else np.full((len(ask), heads, dim), 3, k.dtype), DT[dt]) for _ in range(2)]
    L.Ops.paged_kv_read_int8(*back, *t, dev(ask))
    assert L.take_device_error() == 0
    for got, codes, scales in ((back[0], t[0], t[1]), (back[1], t[2], t[3])):
        got, exp = got.numpy(), ref.read(codes.numpy(), scales.numpy(), ask[:-1])
        # one f32 product, rounded once more to the type
        step = ref.HALF_STEP[got.dtype] + (0 if dt == "f32" else 2.0 ** -24)
        assert (np.abs(ref.widen(got[:-1]) - exp) <= step * np.abs(exp) * (1 + 2.0 ** -20)).all()
        assert (got[-1] == (0x4242 if dt == "bf16" else 3)).all()  # slot -1: as it was


def test_append_many_rows_of_single_tokens():
    # rows of many requests, more than one each to a group of threads, and a step of nothing but padding
    rng = np.random.default_rng(3)
    heads, dim, block, n = 8, 64, 16, 2100
    slots = (rng.permutation(n) * block + rng.integers(0, block, n)).astype(np.int64)
    k, v = (host(rng.standard_normal((n, heads, dim)), "bf16") for _ in range(2))
    _check_append(Cache(n, heads, block, dim), k, v, slots, "bf16")
    _check_append(Cache(2, heads, block, dim), k[:5], v[:5], np.full(5, -1, np.int64), "bf16")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_append_extreme_values(dt):
    heads, dim, block = 2, 32, 16
    rng = np.random.default_rng(5)
    slots = _slots([(0, 4), (2, 5), (16, 20), (30, 34), (8, 9), (1, 2)], block, 12)
    k, v = (rng.standard_normal((len(slots), heads, dim)) for _ in range(2))
    k[0:4] = 0.0  # a new block of zeros
    k[4:7, 0] = 0.0  # zeros into a block that holds values
    k[8, 0, 3], k[9, 1, 4], v[8, 1, :] = np.nan, np.inf, np.nan
    v[11:15] *= 1e-7 if dt == "f16" else 1e-38  # scales below the normal range of f32, or near it
    v[15] *= 3e4 if dt == "f16" else 1e37
    k[16] = 127.0 * 2.0 ** -3 * rng.choice([-1, 1], (heads, dim))  # the largest code itself
    half = np.arange(dim) - 15.5  # quotients exactly between two codes
    v[16] = half * 2.0 ** -4
    v[16, :, 0] = 127 * 2.0 ** -4
    cache = Cache(12, heads, block, dim)
    cache.vs[:] = 2.0 ** -4 if dt != "f32" else cache.vs
    _check_append(cache, host(k, dt), host(v, dt), slots, dt)


def test_append_refuses_slots():
    heads, dim, block = 1, 32, 16
    cache = Cache(4, heads, block, dim)
    k = host(np.random.default_rng(1).standard_normal((3, heads, dim)), "f32")

    def run(slots):
        t = cache.tensors()
        L.Ops.paged_kv_append_int8(*t, dev(k), dev(k), dev(np.array(slots, np.int64)))
        return L.take_device_error(), t[0].numpy(), t[1].numpy()

    err, codes, scales = run([4 * block, 17, 2 ** 40])  # past the pool: skipped, the row between them written
    assert err == 4
    ec, es = ref.append(cache.k, cache.ks, k[1:2], np.array([17]))
    assert np.array_equal(codes, ec) and np.array_equal(scales, es)
    for slots in ([5, 5, 6], [5, 7, 8], [6, 5, 4], [14, 15, 15]):  # twice, a gap, backwards: the block stays as it was
        err, codes, scales = run(slots)
        assert err == 4 and np.array_equal(codes, cache.k) and np.array_equal(scales, cache.ks), slots
    out = [dev(np.full((3, heads, dim), 9, np.float32)) for _ in range(2)]
    L.Ops.paged_kv_read_int8(*out, *cache.tensors(), dev(np.array([64, 3, -5], np.int64)))
    assert L.take_device_error() == 4
    got = out[0].numpy()
    assert (got[[0, 2]] == 9).all() and np.array_equal(got[1], (cache.k[0, :, 3] * cache.ks[0][:, None]).astype(np.float32))


# ---- attention -------------------------------------------------------------------------------


class Attend:
    def __init__(self, rows, lens, nh, heads, dim, block, dt, pad=0, seed=0, sharp=1.0):
        rng = np.random.default_rng(seed)
        n_blocks = sum(-(-n // block) for n in lens) + 2
        self.cache, self.dt, self.scale = Cache(n_blocks, heads, block, dim, seed), dt, 1 / np.sqrt(dim)
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.lens, width = np.array(lens, np.int32), max([-(-n // block) for n in lens] + [1]) + 1
        ids, at = rng.permutation(n_blocks), 0
        self.table = np.full((len(lens), width), -1, np.int32)
        for r, n in enumerate(lens):
            k = -(-n // block)
            self.table[r, :k] = ids[at:at + k]
            at += k
        self.q = host(rng.standard_normal((int(self.starts[-1]) + pad, nh, dim)) * sharp, dt)

    def run(self, out=None):
        c = self.cache
        self.args = [dev(self.q, DT[self.dt]), *c.tensors(), dev(self.table), dev(self.starts), dev(self.lens)]
        out = out or dev(np.full(self.q.shape, 0x4242 if self.dt == "bf16" else 9, self.q.dtype), DT[self.dt])
        L.Ops.paged_attention_int8kv(out, *self.args, self.scale)
        return L.take_device_error(), out.numpy()

    def expect(self):
        c = self.cache
        return ref.attend(self.q, c.k, c.ks, c.v, c.vs, self.table, self.starts, self.lens, self.scale, WEIGHT_STEP[self.dt])

    def check(self, err=0):
        got_err, got = self.run()
        exp, tol = self.expect()
        assert got_err == err
        live = np.arange(len(got)) < self.starts[-1]
        assert (got[~live] == (0x4242 if self.dt == "bf16" else 9)).all()  # rows behind the last request
        g, e = ref.widen(got[live]), exp[live]
        assert (np.isnan(g) == np.isnan(e)).all(), "other outputs are NaN"
        off = np.abs(g - e)[~np.isnan(e)] / tol[live][~np.isnan(e)]
        assert (off <= 1).all(), f"{(off > 1).sum()} of {off.size} beyond the bound, worst {off.max():.3g} of it"
        return got


HEADS = [(12, 2, 128), (32, 8, 128), (16, 16, 64), (10, 10, 80), (7, 1, 16), (3, 1, 256), (40, 1, 96)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nh,heads,dim", HEADS)
def test_attention_decode(nh, heads, dim, dt):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 257, 700, 2, 1000]
    Attend([1] * len(lens), lens, nh, heads, dim, 16, dt, pad=2, seed=nh).check()
    Attend([1] * 3, [300, 1, 129], nh, heads, dim, 64, dt, seed=dim).check()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nh,heads,dim", HEADS)
def test_attention_rows(nh, heads, dim, dt):
    # prompts, chunks after cached tokens, single rows, none
    Attend([37, 1, 0, 64, 5, 130], [37, 90, 50, 64, 133, 300], nh, heads, dim, 32, dt, pad=3, seed=nh + 1).check()


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
def test_attention_blocks(block):
    Attend([1, 40, 3, 200], [513, 255, 256, 457], 4, 2, 128, block, "bf16", seed=block).check()


@pytest.mark.parametrize("rows,lens", [([1], [1]), ([2], [1]), ([5, 3], [3, 0]), ([1, 1], [0, 0]), ([300], [299]), ([0, 0], [7, 9]),
                                       ([20, 1], [0, 5])])
def test_attention_rows_without_keys(rows, lens):
    a = Attend(rows, lens, 6, 2, 64, 16, "bf16", pad=1)
    got = a.check()
    for r, (n, k) in enumerate(zip(rows, lens)):
        empty = max(0, n - k)
        assert (got[a.starts[r]:a.starts[r] + empty] == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,lens", [([1], [20000]), ([3, 1], [5000, 9000]), ([130], [4100])])
def test_attention_long(rows, lens, dt):
    Attend(rows, lens, 12, 2, 128, 64, dt, seed=4).check()


# Rows of a call choose the tiles of its requests, unused ones with them: so many that requests of more than 32 rows go by 128.
def unused(nh):
    return 70000 // nh


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nh,heads,dim", HEADS)
def test_attention_beside_many_unused_rows(nh, heads, dim, dt):
    Attend([37, 1, 0, 64, 5, 130], [37, 90, 50, 64, 133, 300], nh, heads, dim, 32, dt, pad=unused(nh), seed=nh + 1).check()
    Attend([3], [50], nh, heads, dim, 16, dt, pad=unused(nh), seed=nh).check()


@pytest.mark.parametrize("rows,lens", [([300], [299]), ([300, 2], [0, 1]), ([70, 1, 300, 90], [30, 0, 5000, 90]), ([1], [0]), ([150], [9000])])
def test_attention_long_beside_many_unused_rows(rows, lens):
    Attend(rows, lens, 8, 2, 64, 64, "bf16", pad=unused(8), seed=5).check()
    Attend(rows, lens, 8, 2, 64, 64, "f32", pad=unused(8), seed=5).check()


@pytest.mark.parametrize("rows,lens", [([300, 40, 1], [300, 5000, 2000]), ([512], [2500]), ([40, 1, 200], [9000, 30, 200])])
def test_attention_tiles_by_steps(rows, lens):
    # of a call's requests with many rows, those of few steps go by 16 rows and the others by 128
    for dt in ("bf16", "f32"):
        Attend(rows, lens, 32, 4, 64, 64, dt, pad=1, seed=8).check()


def test_attention_many_requests():
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(1, 90, 700)]
    Attend([1] * 700, lens, 4, 2, 64, 16, "bf16").check()
    rows = [int(min(n, x)) for n, x in zip(lens, rng.integers(0, 6, 700))]
    Attend(rows, lens, 4, 2, 64, 16, "f16", pad=40).check()


def test_attention_sharp_and_flat_scores():
    for sharp in (0.0, 30.0):
        Attend([1, 70], [333, 400], 4, 2, 128, 32, "bf16", sharp=sharp).check()
        Attend([1, 70], [333, 400], 4, 2, 128, 32, "f32", sharp=sharp).check()
    a = Attend([1, 70], [333, 400], 4, 2, 128, 32, "f32")
    a.scale = -a.scale
    a.check()


@pytest.mark.parametrize("pad", [0, 17500])
@pytest.mark.parametrize("dt,lo,hi", [("bf16", 1e-30, 1e30), ("f32", 1e-30, 1e30), ("f16", 1e-7, 3e4)])
def test_attention_scales_far_apart(dt, lo, hi, pad):
    # rows of q of very different sizes, blocks of values of very different sizes
    a = Attend([1, 50, 1], [300, 400, 77], 4, 2, 64, 16, dt, pad=pad, seed=2)
    rng = np.random.default_rng(1)
    q = ref.widen(a.q)
    size = np.where(np.arange(len(q)) % 2, lo, hi)[:, None, None]
    a.q = host(np.clip(q * size, -6e4, 6e4) if dt == "f16" else q * size, dt)
    a.cache.ks *= np.float32(1e-3 / hi)
    a.cache.vs *= (10.0 ** rng.integers(-6, 3, a.cache.vs.shape)).astype(np.float32)
    a.cache.vs[::7] = 0.0
    a.check()


@pytest.mark.parametrize("pad", [0, 17500])
def test_attention_non_finite(pad):
    # a block of NaN scale reaches only the rows that see it; a row of q with a NaN only itself
    a = Attend([1, 60, 1], [100, 60, 64], 4, 2, 64, 16, "bf16", pad=pad, seed=6)
    a.cache.vs[a.table[1, 2], 0] = np.nan  # keys 32..47 of request 1, q heads 0 and 1
    a.cache.ks[a.table[1, 3], 1] = np.nan  # keys 48..59, q heads 2 and 3
    a.table[0, 7] = next(b for b in range(len(a.cache.k)) if b not in a.table)
    a.cache.vs[a.table[0, 7]] = a.cache.ks[a.table[0, 7]] = np.nan  # behind the last key of request 0 (100 keys end in block 6)
    q = a.q.copy()
    q[61, 3, 5] = 0x7FC0
    a.q = q
    got = ref.widen(a.check())
    assert np.isnan(got[33:61, :2]).all() and not np.isnan(got[1:33, :2]).any()
    assert np.isnan(got[49:61, 2:]).all() and not np.isnan(got[1:49, 2:]).any()
    assert np.isnan(got[61, 3]).all() and not np.isnan(got[61, :3]).any() and not np.isnan(got[0]).any()


@pytest.mark.parametrize("pad", [0, 17500])
@pytest.mark.parametrize("value", [-1.0, np.inf, -np.inf, np.nan])
def test_attention_scales_that_are_no_scales(value, pad):
    # rows that see such a block are NaN, the others as without it
    for which in ("ks", "vs"):
        a = Attend([1, 60], [100, 60], 4, 2, 64, 16, "bf16", pad=pad, seed=6)
        exp, tol = a.expect()
        getattr(a.cache, which)[a.table[1, 2], 0] = value  # keys 32..47 of request 1, q heads 0 and 1
        err, got = a.run()
        got = ref.widen(got[:61])
        assert err == 0 and np.isnan(got[33:, :2]).all()
        got[33:, :2], exp[33:, :2] = 0, 0
        assert (np.abs(got - exp[:61]) <= tol[:61]).all()


@pytest.mark.parametrize("pad", [0, 17500])
def test_attention_skips_bad_blocks(pad):
    # ids outside the pool: their keys are not attended, and the error word says so
    a = Attend([1, 40], [200, 90], 4, 2, 64, 16, "bf16", pad=pad, seed=7)
    a.table[0, 3], a.table[1, 1], a.table[1, 0] = -1, len(a.cache.k), 2 ** 31 - 1
    a.check(err=4)


def test_attention_refuses_rows_and_lengths():
    a = Attend([1, 2, 3], [50, 60, 70], 4, 2, 64, 16, "bf16", seed=8)
    base = a.run()[1]
    mark = 0x4242

    def run(starts=None, lens=None):
        b = Attend([1, 2, 3], [50, 60, 70], 4, 2, 64, 16, "bf16", seed=8)
        b.starts = b.starts if starts is None else np.array(starts, np.int32)
        b.lens = b.lens if lens is None else np.array(lens, np.int32)
        return b.run()

    err, got = run(lens=[50, 10 ** 6, 70])
    assert err == 4 and np.array_equal(got[[0, 3, 4, 5]], base[[0, 3, 4, 5]]) and (got[1:3] == mark).all()
    err, got = run(lens=[-1, 60, 70])
    assert err == 4 and np.array_equal(got[1:], base[1:]) and (got[0] == mark).all()
    err, got = run(starts=[0, 1, 3, 9])
    assert err == 4 and np.array_equal(got[:3], base[:3]) and (got[3:] == mark).all()


def test_attention_far_blocks():
    # code offsets past 2^32: a pool of 4.5 GB for each of k and v, of which a few blocks are written
    heads, dim, block, n_blocks = 8, 128, 256, 17408
    rng = np.random.default_rng(3)
    t = [L.Tensor((n_blocks, heads, block, dim), L.DataType.I8, **AMD), L.Tensor((n_blocks, heads), L.DataType.F32, **AMD),
         L.Tensor((n_blocks, heads, block, dim), L.DataType.I8, **AMD), L.Tensor((n_blocks, heads), L.DataType.F32, **AMD)]
    n, total = 300, 300
    ids = [n_blocks - 1, 16385]
    slots = np.array([ids[p // block] * block + p % block for p in range(n)], np.int64)
    k, v = (host(rng.standard_normal((n, heads, dim)), "bf16") for _ in range(2))
    L.Ops.paged_kv_append_int8(*t, dev(k, DT["bf16"]), dev(v, DT["bf16"]), dev(slots))
    small = Cache(2, heads, block, dim)
    near = np.arange(n, dtype=np.int64)
    kc, ks = ref.append(small.k, small.ks, k, near)
    vc, vs = ref.append(small.v, small.vs, v, near)
    back = [L.Tensor((n, heads, dim), L.DataType.BF16, **AMD) for _ in range(2)]
    L.Ops.paged_kv_read_int8(*back, *t, dev(slots))
    exp = ref.read(kc, ks, near)
    assert (np.abs(ref.widen(back[0].numpy()) - exp) <= 2.0 ** -7.9 * np.abs(exp)).all()
    for rows in (1, 100):
        q = host(rng.standard_normal((rows, 32, dim)), "bf16")
        starts, lens = np.array([0, rows], np.int32), np.array([total], np.int32)
        out = L.Tensor(q.shape, L.DataType.BF16, **AMD)
        L.Ops.paged_attention_int8kv(out, dev(q, DT["bf16"]), *t, dev(np.array([ids], np.int32)), dev(starts), dev(lens), 0.1)
        exp, tol = ref.attend(q, kc, ks, vc, vs, np.array([[0, 1]]), starts, lens, 0.1, WEIGHT_STEP["bf16"])
        assert (np.abs(ref.widen(out.numpy()) - exp) <= tol).all()
    assert L.take_device_error() == 0


def test_attention_repeats_bit_for_bit():
    a = Attend([1, 1, 200, 9], [9000, 333, 1200, 800], 12, 2, 128, 64, "bf16", seed=11)
    first = a.run()[1]
    for _ in range(3):
        assert np.array_equal(a.run()[1], first)


# ---- a run of them together ------------------------------------------------------------------


class Server:
    """Requests that are served step by step: lengths in, attention out, one layer."""

    def __init__(self, requests, nh, heads, dim, block, n_blocks, rows, dt):
        self.nh, self.heads, self.dim, self.block, self.rows, self.dt = nh, heads, dim, block, rows, dt
        width = n_blocks
        I32, I64, T = L.DataType.I32, L.DataType.I64, DT[dt]
        new = lambda shape, d: L.Tensor(shape, d, **AMD)
        self.cache = [new((n_blocks, heads, block, dim), L.DataType.I8), new((n_blocks, heads), L.DataType.F32),
                      new((n_blocks, heads, block, dim), L.DataType.I8), new((n_blocks, heads), L.DataType.F32)]
        for t in self.cache:
            t.load(np.zeros(t.shape(), np.int8 if t.dtype() == L.DataType.I8 else np.float32).ctypes.data)
        self.table, self.ring, self.state = dev(np.full((requests, width), -1, np.int32)), dev(np.arange(n_blocks, dtype=np.int32)), dev(np.array([0, n_blocks]))
        self.slots, self.pos, self.starts = new((rows,), I64), new((rows,), I64), new((requests + 1,), I32)
        self.old, self.new_ = new((requests,), I32), new((requests,), I32)
        self.q, self.k, self.v = new((rows, nh, dim), T), new((rows, heads, dim), T), new((rows, heads, dim), T)
        self.q_rot, self.k_rot, self.out = new((rows, nh, dim), T), new((rows, heads, dim), T), new((rows, nh, dim), T)

    def load(self, old, new, q, k, v):
        for t, a in ((self.old, np.array(old, np.int32)), (self.new_, np.array(new, np.int32)), (self.q, q), (self.k, k), (self.v, v)):
            a = np.ascontiguousarray(a)
            t.load(a.ctypes.data)

    def step(self):
        L.Ops.paged_tables(self.table, self.slots, self.pos, self.starts, self.state, self.old, self.new_, self.ring, self.state, self.block)
        L.Ops.rope_qk(self.q_rot, self.q, self.k_rot, self.k, self.pos, 1e6)
        L.Ops.paged_kv_append_int8(*self.cache, self.k_rot, self.v, self.slots)
        L.Ops.paged_attention_int8kv(self.out, self.q_rot, *self.cache, self.table, self.starts, self.new_, 1 / np.sqrt(self.dim))


@pytest.mark.parametrize("dt,captured", [("bf16", False), ("bf16", True), ("f32", False)])
def test_server_steps(dt, captured):
    # prompts, generated tokens, a request that ends and one that takes its place, speculative rows taken back
    requests, nh, heads, dim, block, n_blocks, rows = 4, 6, 2, 64, 16, 40, 170
    s = Server(requests, nh, heads, dim, block, n_blocks, rows, dt)
    steps = [[60, 17, 0, 80], [61, 18, 0, 81], [62, 23, 33, 0], [63, 19, 34, 40], [64, 24, 35, 41], [0, 25, 36, 200]]
    rng = np.random.default_rng(0)
    r_table, r_ring, r_state = np.full((requests, n_blocks), -1, np.int32), np.arange(n_blocks, dtype=np.int32), np.array([0, n_blocks])
    kc, vc = (np.zeros((n_blocks, heads, block, dim), np.int8) for _ in range(2))
    ks, vs = (np.zeros((n_blocks, heads), np.float32) for _ in range(2))
    graph, old = None, [0] * requests
    for new in steps:
        q, k, v = (host(rng.standard_normal((rows, h, dim)), dt) for h in (nh, heads, heads))
        s.load(old, new, q, k, v)
        if captured:
            if graph is None:
                graph = L.Graph.capture()
                s.step()
                graph.end()
            graph.launch()
        else:
            s.step()
        assert L.take_device_error() == 0
        r_table, r_ring, r_state, slots, pos, starts = ref.tables(r_table, r_ring, r_state, old, new, block, rows)
        for t, e in ((s.table, r_table), (s.ring, r_ring), (s.state, r_state), (s.slots, slots), (s.pos, pos), (s.starts, starts)):
            assert np.array_equal(t.numpy(), e)
        kc, ks = ref.append(kc, ks, s.k_rot.numpy(), slots)
        vc, vs = ref.append(vc, vs, v, slots)
        for t, e in zip(s.cache, (kc, ks, vc, vs)):
            assert np.array_equal(t.numpy(), e)
        exp, tol = ref.attend(s.q_rot.numpy(), kc, ks, vc, vs, r_table, starts, new, 1 / np.sqrt(dim), WEIGHT_STEP[dt])
        n = starts[-1]
        assert (np.abs(ref.widen(s.out.numpy()[:n]) - exp[:n]) <= tol[:n]).all()
        old = new


def test_two_graphs_and_eager_calls_share_the_scratch():
    a = Attend([1, 1], [6000, 900], 12, 2, 128, 64, "bf16", seed=20)
    b = Attend([2], [7000], 12, 2, 128, 64, "bf16", seed=21)
    c = Attend([150], [2000], 12, 2, 128, 64, "bf16", seed=22)
    want, graphs = [x.run()[1] for x in (a, b, c)], []
    for x in (a, b):
        x.out = L.Tensor(x.q.shape, DT["bf16"], **AMD)
        g = L.Graph.capture()
        L.Ops.paged_attention_int8kv(x.out, *x.args, x.scale)
        graphs.append(g.end())
    for _ in range(3):
        for x in (a, b):
            x.out.load(np.zeros(x.q.shape, np.uint16).ctypes.data)
        graphs[0].launch()
        graphs[1].launch()
        assert np.array_equal(c.run()[1], want[2])
        assert np.array_equal(a.out.numpy(), want[0]) and np.array_equal(b.out.numpy(), want[1])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_append_rounds_older_codes_as_exact_quotients(dt):
    # every code at many ratios of scales, ratios of small whole numbers (ties) and others next to them among them
    rng = np.random.default_rng(8)
    heads, dim, block, n = 8, 256, 16, 64
    cache = Cache(n, heads, block, dim)
    cache.k[:, :, :] = (np.arange(dim) - 128).clip(-127, 127).astype(np.int8)
    ratio = rng.choice([2.0, 4.0, 6.0, 1.5, 3.0, 10.0, 1.0 + 2.0 ** -20, 1.25, 254.0], (n, heads)) * rng.choice([1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -23], (n, heads))
    cache.ks = (2.0 ** rng.integers(-20, 20, (n, heads)) * rng.choice([1.0, 1.1, 1.7], (n, heads))).astype(np.float32)
    k = np.zeros((n, heads, dim))
    k[:, :, 0] = 127.0 * cache.ks * ratio
    slots = (np.arange(n) * block + 15).astype(np.int64)
    _check_append(cache, host(k, dt), host(k, dt), slots, dt)
