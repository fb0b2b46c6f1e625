"""The KV cache in blocks without a GPU: refusals of its entry points, and the reference the GPU tests compare with."""
import numpy as np
import pytest

import paged_ref as ref
from test_abi import _run

CACHE = "I8, I32, I64, BF = L.DataType.I8, L.DataType.I32, L.DataType.I64, L.DataType.BF16; " \
        "kc, ks, vc, vs = t((4,2,16,32), I8), t((4,2)), t((4,2,16,32), I8), t((4,2)); k = t((3,2,32)); s = t((3,), I64); "
APPEND = CACHE + "L.Ops.paged_kv_append_int8({})"
READ = CACHE + "L.Ops.paged_kv_read_int8({})"
ATTEND = CACHE + "q, o, tab, st, ln = t((3,4,32)), t((3,4,32)), t((2,2), I32), t((3,), I32), t((2,), I32); " \
                 "L.Ops.paged_attention_int8kv({}, 0.1)"
TABLES = CACHE + "tab, st, ln, l2, ring, fi, fo, sl, po = t((2,2), I32), t((3,), I32), t((2,), I32), t((2,), I32), t((4,), I32), " \
                 "t((2,), I64), t((2,), I64), t((3,), I64), t((3,), I64); L.Ops.paged_tables({})"


@pytest.mark.parametrize("code,message", [
    (APPEND.format("kc, ks, vc, vs, k, k, s"), "Unsupported device"),
    (APPEND.format("kc, ks, vc, vs, k, t((3,2,32), BF), s"), "Datatypes mismatch"),
    (APPEND.format("kc, ks, vc, vs, k, t((4,2,32)), s"), "Shapes mismatch"),
    (APPEND.format("kc, ks, vc, vs, t((3,1,32)), t((3,1,32)), s"), "kv head shape mismatch"),
    (APPEND.format("kc, ks, vc, vs, k, k, t((2,), I64)"), "one slot per row"),
    (APPEND.format("kc, ks, vc, vs, k, k, t((3,), I32)"), "slots must be INT64"),
    (APPEND.format("kc, ks, vc, vs, t((3,2,32), I32), t((3,2,32), I32), s"), "Unsupported data type"),
    (APPEND.format("k, ks, vc, vs, k, k, s"), "cache codes must be INT8"),
    (APPEND.format("kc, t((4,2), BF), vc, vs, k, k, s"), "cache scales must be F32"),
    (APPEND.format("kc, t((4,3)), vc, t((4,3)), k, k, s"), "scale cache shape mismatch"),
    (APPEND.format("kc, ks, t((5,2,16,32), I8), vs, k, k, s"), "Shapes mismatch"),
    (APPEND.format("t((4,2,24,32), I8), ks, t((4,2,24,32), I8), vs, k, k, s"), "block must be a power of two in [16, 256]"),
    (APPEND.format("t((4,2,16,40), I8), ks, t((4,2,16,40), I8), vs, t((3,2,40)), t((3,2,40)), s"), "head_dim must be a multiple of 16"),
    (APPEND.format("t((4,2,16,272), I8), ks, t((4,2,16,272), I8), vs, t((3,2,272)), t((3,2,272)), s"), "head_dim must be a multiple of 16"),
    (APPEND.format("kc, ks, kc, vs, k, k, s"), "caches must not overlap"),
    (APPEND.format("kc.permute(0,1,3,2).permute(0,1,3,2).slice(3,0,16), ks, kc.slice(3,0,16), vs, k, k, s"), "must be contiguous"),
    (READ.format("k, t((3,2,32)), kc, ks, vc, vs, s"), "Unsupported device"),
    (READ.format("k, k, kc, ks, vc, vs, s"), "k and v must not overlap"),
    (ATTEND.format("o, q, kc, ks, vc, vs, tab, st, ln"), "Unsupported device"),
    (ATTEND.format("o, t((3,4,16)), kc, ks, vc, vs, tab, st, ln"), "Shapes mismatch"),
    (ATTEND.format("t((3,4,16)), t((3,4,16)), kc, ks, vc, vs, tab, st, ln"), "head_dim mismatch"),
    (ATTEND.format("o, q, t((0,2,16,32), I8), t((0,2)), t((0,2,16,32), I8), t((0,2)), tab, st, ln"), "the cache has no blocks"),
    (ATTEND.format("t((3,3,32)), t((3,3,32)), kc, ks, vc, vs, tab, st, ln"), "divisible by kv_head"),
    (ATTEND.format("t((3,4,32), BF), q, kc, ks, vc, vs, tab, st, ln"), "Datatypes mismatch"),
    (ATTEND.format("o, q, kc, ks, vc, vs, t((2,2), I64), st, ln"), "must be INT32"),
    (ATTEND.format("o, q, kc, ks, vc, vs, t((2,), I32), st, ln"), "block_table [requests, width]"),
    (ATTEND.format("o, q, kc, ks, vc, vs, tab, st, st"), "a length per request"),
    (ATTEND.format("o, q, kc, ks, vc, vs, tab, ln, ln"), "requests + 1 elements"),
    (ATTEND.format("q, q, kc, ks, vc, vs, tab, st, ln"), "must not overlap q"),
    (TABLES.format("tab, sl, po, st, fo, ln, l2, ring, fi, 16"), "Unsupported device"),
    (TABLES.format("tab, sl, po, st, fi, ln, l2, ring, fi, 16"), "Unsupported device"),
    (TABLES.format("tab, sl, po, st, fo, ln, l2, ring, fi, 20"), "block must be a power of two"),
    (TABLES.format("tab, sl, po, ln, fo, ln, l2, ring, fi, 16"), "requests + 1 elements"),
    (TABLES.format("tab, sl, t((4,), I64), st, fo, ln, l2, ring, fi, 16"), "the same length"),
    (TABLES.format("tab, sl, po, st, fo, ln, st, ring, fi, 16"), "one old and one new length"),
    (TABLES.format("tab, st, po, st, fo, ln, l2, ring, fi, 16"), "must be INT64"),
    (TABLES.format("tab, sl, sl, st, fo, ln, l2, ring, fi, 16"), "outputs must not overlap"),
    (TABLES.format("tab, sl, po, st, fo, ln, l2, tab.view(4), fi, 16"), "outputs must not overlap"),
    (TABLES.format("tab, sl, po, st, fo, tab.view(4).slice(0,0,2), l2, ring, fi, 16"), "must not overlap inputs"),
    (TABLES.format("t((8193,1), I32), sl, po, t((8194,), I32), fo, t((8193,), I32), t((8193,), I32), ring, fi, 16"), "at most 8192 requests"),
    (TABLES.format("tab, sl, po, st, t((3,), I64), ln, l2, ring, fi, 16"), "the ring's state is (head, tail)"),
])
def test_refusals(code, message):
    r = _run(code)
    assert r.returncode != 0 and "RETURNED" not in r.stdout
    assert message in r.stderr and "[ERROR]" in r.stderr, r.stderr[-2000:]


def test_reference_attention_against_a_direct_sum():
    # two requests, two kv heads of two q heads, blocks of 16: each output by loops over the definition
    rng = np.random.default_rng(0)
    heads, dim, block = 2, 16, 16
    k, v = (rng.integers(-127, 128, (5, heads, block, dim)).astype(np.int8) for _ in range(2))
    ks, vs = (rng.uniform(0.01, 0.03, (5, heads)).astype(np.float32) for _ in range(2))
    table, starts, lens = np.array([[3, 1], [4, 0]], np.int32), np.array([0, 3, 4], np.int32), np.array([20, 17], np.int32)
    q = rng.standard_normal((4, 4, dim)).astype(np.float32)
    out, _ = ref.attend(q, k, ks, v, vs, table, starts, lens, 0.25, 0.0)
    for r in range(2):
        for t in range(starts[r], starts[r + 1]):
            last = lens[r] - (starts[r + 1] - t)
            for h in range(4):
                w, acc, total = [], np.zeros(dim), 0.0
                for key in range(last + 1):
                    b, o = table[r, key // block], key % block
                    w.append(0.25 * float(ks[b, h // 2]) * float(np.dot(q[t, h].astype(float), k[b, h // 2, o].astype(float))))
                for key, s in enumerate(w):
                    b, o, p = table[r, key // block], key % block, np.exp(s - max(w))
                    acc, total = acc + p * float(vs[b, h // 2]) * v[b, h // 2, o], total + p
                assert np.allclose(out[t, h], acc / total, rtol=1e-12, atol=1e-12)


def test_reference_tables_and_append():
    got = ref.tables(np.array([[5, -1, -1], [2, 8, -1]], np.int32), np.array([1, 3, 9, 0], np.int32), [2, 4], [10, 20], [33, 0], 16, 24)
    table, ring, state, slots, pos, starts = got
    assert state.tolist() == [4, 6] and ring.tolist() == [2, 8, 9, 0] and table[0].tolist() == [5, 9, 0]
    assert starts.tolist() == [0, 23, 23] and pos[:23].tolist() == list(range(10, 33)) and slots[23] == -1
    assert slots[:7].tolist() == [90, 91, 92, 93, 94, 95, 144] and slots[22] == 0
    codes, scales = np.full((1, 1, 16, 16), 100, np.int8), np.full((1, 1), 1.0, np.float32)
    c, s = ref.append(codes, scales, np.full((2, 1, 16), 254.0, np.float32), np.array([3, 4]))
    assert s[0, 0] == 2.0 and (c[0, 0, :3] == 50).all() and (c[0, 0, 3:5] == 127).all() and (c[0, 0, 5:] == 100).all()
    c, s = ref.append(codes, scales, np.full((1, 1, 16), -0.5, np.float32), np.array([0]))  # a new block: the old scale is gone
    assert s[0, 0] == np.float32(0.5) / np.float32(127) and (c[0, 0, 0] == -127).all()
