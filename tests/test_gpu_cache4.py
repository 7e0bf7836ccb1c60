"""The 4-bit key / value cache (include/we_cache4.h) on the GPU against its plain 64-bit form (cache4_lib)."""
import numpy as np
import pytest

import cache4_lib as C
import we

pytestmark = pytest.mark.gpu
TYPES = [we.F32, we.F16, we.BF16]
NAN_BITS = {we.F32: np.float32(np.nan), we.F16: np.uint16(0x7e00), we.BF16: np.uint16(0x7fc0)}


@pytest.fixture
def scope(graph):
    """buffers made in the test go back after it"""
    mark = graph.mark()
    yield graph
    graph.sync()
    graph.release(mark)


def ints(graph, values):
    return graph.buffer(np.asarray(values, np.int32))


def rows(rng, batch, tokens, heads, dim, dtype, stride=0, spread=1.0):
    """(values [batch, tokens, heads, dim], the array of rows `stride` apart with NaN between them)"""
    x = C.store(rng.standard_normal((batch, tokens, heads, dim)) * spread, dtype)
    st = stride or heads * dim
    a = np.full((batch * tokens, st), NAN_BITS[dtype], C.NP[dtype])
    a[:, :heads * dim] = x.reshape(batch * tokens, heads * dim)
    return C.value(x, dtype), a


def filled(rng, batch, kv, dim, cap, lens, spread=1.0, offset=0.5):
    """a cache whose first lens[b] slots hold K and V rows and the rest anything"""
    c = C.Cache(batch, kv, dim, cap, fill=rng)
    for b, n in enumerate(lens):
        n = min(n, cap)
        if n > 0:
            k, v = ((rng.standard_normal((n, kv, dim)) * spread + rng.standard_normal((kv, dim)) * offset) for _ in range(2))
            c.put(b, 0, k, v)
    return c


# ------------------------------------------------------------------------------------------------- append and load

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,kv,dim,cap,tokens,lens,counts,stride", [
    (1, 1, 64, 64, 1, [0], None, 0),                       # the first token of the smallest cache
    (3, 2, 128, 192, 1, [5, 0, 191], None, 0),             # a decode step, the last sequence's last slot
    (2, 3, 192, 128, 7, [120, 3], None, 1024),             # a row stride; one sequence runs out of slots
    (2, 1, 256, 64, 5, [64, -3], [5, 9], 0),               # full; a length and a count out of range
    (4, 2, 128, 320, 129, [0, 17, 64, 100], [129, 0, 1, 77], 0),  # a padded batch of prompts, several workgroups
])
def test_append_then_load(scope, dtype, batch, kv, dim, cap, tokens, lens, counts, stride):
    g, rng = scope, np.random.default_rng(batch * 1000 + dim + tokens)
    k, ka = rows(rng, batch, tokens, kv, dim, dtype, stride)
    v, va = rows(rng, batch, tokens, kv, dim, dtype, stride)
    c = C.Cache(batch, kv, dim, cap, fill=rng)
    h = c.handle(g)
    n = [tokens if counts is None else min(max(x, 0), tokens) for x in counts or lens]
    start = [min(max(x, 0), cap) for x in lens]
    seen = [x + 11 for x in start]
    pos, weight = (rng.integers(0, 99, (batch, kv, cap)).astype(t) for t in (np.int32, np.float32))
    pb, wb, lb, sb = g.buffer(pos), g.buffer(weight), ints(g, lens), ints(g, seen)
    old = ints(g, lens)
    g.cache4_append(h, tokens, dtype, g.buffer(ka), g.buffer(va), lb, lb, stride, stride,
                    None if counts is None else ints(g, counts), sb, sb, pb, wb)
    for b in range(batch):
        m = min(n[b], cap - start[b])
        c.put(b, start[b], k[b, :m], v[b, :m])
        pos[b, :, start[b]:start[b] + m] = seen[b] + np.arange(m)
        weight[b, :, start[b]:start[b] + m] = 0
    assert np.array_equal(g.read(h.data), c.bytes)  # every code and scale, and nothing else
    assert np.array_equal(g.read(pb, dtype=np.int32), pos.reshape(-1))
    assert np.array_equal(g.read(wb, dtype=np.float32), weight.reshape(-1))
    assert g.read(lb, dtype=np.int32).tolist() == [min(s + m, cap) for s, m in zip(start, n)]
    assert g.read(sb, dtype=np.int32).tolist() == [s + m for s, m in zip(seen, n)]

    ko, vo = (g.buffer(np.full_like(ka, 7)) for _ in range(2))
    g.cache4_load(h, tokens, dtype, ko, vo, first=old, lens=lb, k_stride=stride, v_stride=stride)
    for got, which in ((ko, 0), (vo, 1)):
        want = np.full_like(ka, 7).reshape(batch, tokens, -1)
        for b in range(batch):
            m = min(n[b], cap - start[b])
            x = c.values(b, cap)[which][:, start[b]:start[b] + m].swapaxes(0, 1)
            want[b, :m, :kv * dim] = C.store(x, dtype).reshape(m, kv * dim)
        assert np.array_equal(g.read(got, dtype=C.NP[dtype]), want.reshape(-1))


def test_append_special_values(scope):
    g, rng = scope, np.random.default_rng(5)
    x = rng.standard_normal((1, 8, 1, 128)).astype(np.float32)
    x[0, 0, 0, 3] = np.nan             # one group of NaN, its neighbour untouched
    x[0, 1, 0, 64:] = 2.5              # a constant group: scale 0
    x[0, 2, 0, 7], x[0, 2, 0, 9] = np.inf, -1e30
    x[0, 3] *= 1e-7                    # subnormal scales
    x[0, 4] = 0.0
    x[0, 5] *= 1e-12                   # scale rounds to 0
    x[0, 6] *= 20000
    x[0, 7] = np.arange(128) % 16 / 2 + 0.25  # ties: the scale is 0.5, every value a half above a code with minimum 0.25
    c = C.Cache(1, 1, 128, 64)
    h = c.handle(g)
    lens = ints(g, [0])
    b = g.buffer(x)
    g.cache4_append(h, 8, we.F32, b, b, lens, lens)
    c.put(0, 0, x[0].astype(np.float64), x[0].astype(np.float64))
    assert np.array_equal(g.read(h.data), c.bytes)
    k, _ = c.values(0, 8)
    assert np.isnan(k[0, 0, :64]).all() and not np.isnan(k[0, 0, 64:]).any()
    # from -65504 to 65504: the scale 8733.9 is 8736 as f16 (steps of 8), and -65504 + 15 * 8736 = 65536
    assert (k[0, 1, 64:] == 2.5).all() and k[0, 2, 7] == 65536 and k[0, 2, 9] == -65504 and (k[0, 5] == 0).all()


def test_append_no_tokens_and_no_seen(scope):
    g, c = scope, C.Cache(2, 1, 64, 64)
    h, lens, out = c.handle(g), ints(g, [3, 70]), ints(g, [-1, -1])
    g.cache4_append(h, 0, we.F16, None, None, lens, out)
    assert g.read(out, dtype=np.int32).tolist() == [3, 64]
    x, pos = g.buffer(np.zeros((2, 2, 64), np.float32)), ints(g, np.full((2, 1, 64), -1))
    g.cache4_append(h, 2, we.F32, x, x, lens, out, pos=pos)
    p = g.read(pos, dtype=np.int32).reshape(2, 64)
    assert p[0, 3:5].tolist() == [3, 4] and (np.delete(p[0], [3, 4]) == -1).all() and (p[1] == -1).all()


# ------------------------------------------------------------------------------------------------------- attention

def check_attention(g, c, q, qa, lens, counts, causal, dtype, q_stride=0, out_stride=0, max_len=0, track=True, handle=None):
    b, tokens, heads, dim = q.shape
    rng = np.random.default_rng(1)
    h = handle or c.handle(g)
    st = out_stride or heads * dim
    before = np.full((b * tokens, st), 3, C.NP[dtype])
    ob = g.buffer(before)
    weight = rng.uniform(0, 2, (b, c.kv, c.cap)).astype(np.float32)
    wi, wo = g.buffer(weight), g.buffer(np.full_like(weight, -5))
    g.cache4_attention(h, tokens, heads, causal, dtype, g.buffer(qa), ints(g, lens), ob, q_stride, out_stride,
                       None if counts is None else ints(g, counts), max_len, wi if track else None, wo if track else None)
    lens = [min(x, max_len or c.cap) for x in lens]
    want, received, bounds = C.attention(c, q, lens, counts or [tokens] * b, causal)
    got = g.read(ob, dtype=C.NP[dtype]).reshape(b * tokens, st)
    assert np.array_equal(got[:, heads * dim:], before[:, heads * dim:])  # between the rows
    got = got[:, :heads * dim].reshape(q.shape)
    alone = np.isnan(want).all((2, 3))
    assert (got[alone] == 3).all()
    err, tol = np.abs(C.value(got, dtype) - want), C.tolerance(want, bounds, dtype)
    assert np.isfinite(err[~alone]).all()
    worst = (err / np.maximum(tol, 1e-300))[~alone]
    assert worst.size == 0 or worst.max() <= 1, worst.max()
    if track:
        w = g.read(wo, dtype=np.float32).reshape(weight.shape)
        for i, n in enumerate(lens):
            n = max(0, min(n, c.cap))
            assert (w[i, :, n:] == -5).all()
            off = np.abs(w[i, :, :n] - (weight[i, :, :n] + received[i, :, :n]))
            tol = C.weight_tolerance(received, bounds)[i, :, :n] + np.abs(w[i, :, :n]) * 2.0 ** -24
            assert (off <= tol).all(), (off / tol).max()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,heads,kv,dim,cap,tokens,lens,counts,causal", [
    (1, 1, 1, 64, 64, 1, [1], None, True),                      # one head, one slot
    (1, 7, 1, 128, 64, 1, [64], None, True),                    # a full cache of one tile
    (2, 28, 4, 128, 192, 1, [131, 65], None, True),             # grouped heads, ragged
    (3, 8, 8, 64, 320, 1, [0, 63, 300], None, False),           # an empty sequence; no shared heads
    (1, 16, 1, 192, 1088, 1, [1030], None, True),               # 16 rows; dim 192; a ragged end
    (2, 24, 2, 256, 256, 1, [200, 129], None, True),            # 12 rows a kv head, dim 256
    (2, 6, 2, 128, 256, 5, [200, 3], None, True),               # more queries than slots: rows that see nothing
    (2, 10, 2, 128, 256, 5, [200, 3], [3, 0], True),            # a padded batch
    (1, 17, 1, 128, 192, 1, [150], None, False),                # a row over a tile of 16
    (1, 8, 2, 64, 256, 33, [250], None, True),                  # a piece of a prompt
    (2, 4, 4, 128, 384, 130, [380, 130], [130, 100], True),     # a prompt from the start
    (1, 10, 2, 192, 128, 40, [100], None, False),
    (1, 8, 1, 256, 192, 41, [170], None, True),
])
def test_attention(scope, dtype, batch, heads, kv, dim, cap, tokens, lens, counts, causal):
    rng = np.random.default_rng(heads * 100 + dim + tokens)
    c = filled(rng, batch, kv, dim, cap, lens)
    q, qa = rows(rng, batch, tokens, heads, dim, dtype)
    check_attention(scope, c, q, qa, lens, counts, causal, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,length", [(1, 4001), (1, 16384), (3, 9000), (20, 5000)])
def test_attention_over_a_long_cache(scope, dtype, tokens, length):
    rng = np.random.default_rng(length)
    c = filled(rng, 1, 2, 128, 16384, [length])
    q, qa = rows(rng, 1, tokens, 4, 128, dtype)
    check_attention(scope, c, q, qa, [length], None, True, dtype)
    check_attention(scope, c, q, qa, [length], None, True, dtype, max_len=length, track=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides_and_max_len(scope, dtype):
    rng = np.random.default_rng(3)
    c = filled(rng, 2, 2, 64, 256, [200, 90])
    q, qa = rows(rng, 2, 4, 6, 64, dtype, stride=648)
    check_attention(scope, c, q, qa, [200, 90], None, True, dtype, q_stride=648, out_stride=392)
    check_attention(scope, c, q, qa, [200, 90], None, True, dtype, q_stride=648, max_len=100)  # read as 100
    check_attention(scope, c, q, qa, [1 << 30, -5], None, False, dtype, q_stride=648, max_len=150)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["small_v", "outlier_v", "constant", "sharp", "zero_q", "large_q", "late_max", "tiny_q"])
def test_attention_value_ranges(scope, dtype, kind):
    """Where f16 operands could run out of range: V far below and above 1, scales far apart, scores far apart."""
    rng = np.random.default_rng(len(kind))
    n, kv, dim, heads = 330, 2, 128, 6
    k, v = rng.standard_normal((2, n, kv, dim))
    q = rng.standard_normal((1, 2, heads, dim))
    if kind == "small_v":
        v *= 1e-5
    elif kind == "outlier_v":
        v *= 1e-3
        v[200] *= 1e7
    elif kind == "constant":
        v[:] = 1.5
        k[:, :, :64] = 0.25
    elif kind == "sharp":
        q *= 40
    elif kind == "zero_q":
        q[0, 0] = 0
    elif kind == "large_q":
        q *= 1e4
        k *= 1e-4  # subnormal scales
    elif kind == "late_max":
        k[300] = 8 * q[0, 1, 0]
    else:
        q *= 1e-4 if dtype == we.F16 else 1e-30
    c = C.Cache(1, kv, dim, 384, fill=rng)
    c.put(0, 0, k, v)
    qs = C.store(q, dtype)
    check_attention(scope, c, C.value(qs, dtype), qs, [n], None, True, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_nan_and_inf_stay_where_they_are(scope, dtype):
    """NaN in a slot reaches the rows that see it and no others; a NaN or infinite query its own row."""
    g, rng = scope, np.random.default_rng(9)
    n, heads = 100, 4
    c = filled(rng, 1, 2, 128, 128, [n])
    clean = C.Cache(1, 2, 128, 128)
    clean.bytes[:] = c.bytes
    c.vs[0, 1, 97] = c.ks[0, 1, 97] = 0x7e007e00
    q, qa = rows(rng, 1, 6, heads, 128, dtype)  # rows 0 .. 5 see 95 .. 100 slots
    ref = check_attention(g, clean, q, qa, [n], None, True, dtype)
    got = g.buffer(qa.nbytes)
    wo = g.buffer(2 * 128 * 4)
    g.cache4_attention(c.handle(g), 6, heads, True, dtype, g.buffer(qa), ints(g, [n]), got, weight_out=wo)
    a = g.read(got, dtype=C.NP[dtype]).reshape(ref.shape)
    assert np.array_equal(a[:, :, :2], ref[:, :, :2]) and np.array_equal(a[:, :3, 2:], ref[:, :3, 2:])
    assert np.isnan(C.value(a[:, 3:, 2:], dtype)).all()
    assert np.isfinite(g.read(wo, dtype=np.float32).reshape(2, 128)[0]).all()
    qa2 = qa.reshape(6, heads, 128).copy()
    qa2[1, 1, 5], qa2[2, 0, 5] = NAN_BITS[dtype], C.store(np.inf, dtype)
    g.cache4_attention(clean.handle(g), 6, heads, True, dtype, g.buffer(qa2), ints(g, [n]), got)
    a = g.read(got, dtype=C.NP[dtype]).reshape(6, heads, 128)
    bad = np.zeros((6, heads), bool)
    bad[1, 1] = bad[2, 0] = True
    assert np.array_equal(a[~bad], ref.reshape(6, heads, 128)[~bad])
    assert np.isnan(C.value(a[bad], dtype)).all()


def test_attention_repeats_bit_for_bit(scope):
    g, rng = scope, np.random.default_rng(12)
    c = filled(rng, 2, 2, 128, 4096, [4000, 1777])
    q, qa = rows(rng, 2, 1, 8, 128, we.BF16)
    h, lens, qb = c.handle(g), ints(g, [4000, 1777]), g.buffer(qa)
    outs = []
    for _ in range(3):
        o, w = g.buffer(qa.nbytes), g.buffer(2 * 2 * 4096 * 4)
        g.cache4_attention(h, 1, 8, True, we.BF16, qb, lens, o, weight_out=w)
        outs.append((g.read(o), g.read(w)))
    assert all(np.array_equal(a, b) for x in outs[1:] for a, b in zip(x, outs[0]))


def test_weight_adds_in_place_and_from_nothing(scope):
    g, rng = scope, np.random.default_rng(13)
    c = filled(rng, 1, 1, 64, 64, [40])
    q, qa = rows(rng, 1, 1, 4, 64, we.F16)
    h, lens, qb, o = c.handle(g), ints(g, [40]), g.buffer(qa), g.buffer(qa.nbytes)
    w = g.buffer(np.full(64, np.nan, np.float32))
    g.cache4_attention(h, 1, 4, True, we.F16, qb, lens, o, weight_out=w)
    one = g.read(w, dtype=np.float32)
    assert abs(one[:40].sum() - 4) < 1e-4 and np.isnan(one[40:]).all()
    g.cache4_attention(h, 1, 4, True, we.F16, qb, lens, o, weight=w, weight_out=w)
    assert np.array_equal(g.read(w, dtype=np.float32)[:40], one[:40] + one[:40])


def test_regions_past_32_bit_offsets(scope):
    """A cache of 4.8 GB whose last sequence and head lie behind every 32-bit byte offset of their region's start."""
    g, rng = scope, np.random.default_rng(14)
    batch, kv, dim, cap = 2, 8, 128, 1 << 21
    h = we.Cache4(g, batch, kv, dim, cap, data=g.buffer(batch * kv * cap * 144))
    lens, out = ints(g, [0, 0]), ints(g, [0, 0])
    k, ka = rows(rng, batch, 70, kv, dim, we.F16)
    v, va = rows(rng, batch, 70, kv, dim, we.F16)
    g.cache4_append(h, 70, we.F16, g.buffer(ka), g.buffer(va), lens, out)
    c = C.Cache(batch, kv, dim, 128)
    for b in range(batch):
        c.put(b, 0, k[b], v[b])
    q, qa = rows(rng, batch, 1, kv, dim, we.F16)
    c.cap, o = 128, g.buffer(qa.nbytes)
    g.cache4_attention(h, 1, kv, True, we.F16, g.buffer(qa), out, o)
    want, _, bounds = C.attention(c, q, [70, 70], [1, 1], True)
    got = C.value(g.read(o, dtype=np.uint16).reshape(q.shape), we.F16)
    assert (np.abs(got - want) <= C.tolerance(want, bounds, we.F16)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv,tokens,lens", [
    (128, 8, 2, 1, [4100, 3, 0, 2100, 64]),      # shares of sequences of very different length, one of them empty
    (64, 32, 8, 1, [3000] * 7),                  # rows of 4 heads; as many shares as fit
    (256, 12, 2, 2, [2200, 2177]),               # 12 rows
    (192, 5, 1, 3, [5000]),                      # 15 rows
    (128, 6, 2, 9, [2500, 2049]),                # 27 rows: two blocks a wave, shared out
    (256, 5, 1, 8, [2300]),                      # 40 rows in three row blocks, shared out
])
def test_attention_shared_out(scope, dtype, dim, heads, kv, tokens, lens):
    rng = np.random.default_rng(dim + heads)
    cap = (max(lens) + 63) // 64 * 64
    c = filled(rng, len(lens), kv, dim, cap, lens)
    q, qa = rows(rng, len(lens), tokens, heads, dim, dtype)
    check_attention(scope, c, q, qa, lens, None, True, dtype)
    check_attention(scope, c, q, qa, lens, None, False, dtype, max_len=max(lens) - 1)  # an odd row of scores


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_few_rows_without_room_for_their_scores(scope, dtype):
    """64 heads over a capacity of 2^20 + 64 slots: their scores would take more than 256 MB."""
    g, rng = scope, np.random.default_rng(18)
    cap = (1 << 20) + 64
    h = we.Cache4(g, 1, 8, 64, cap, data=g.buffer(8 * cap * 72))
    lens = ints(g, [700])
    k, ka = rows(rng, 1, 700, 8, 64, we.F16)
    v, va = rows(rng, 1, 700, 8, 64, we.F16)
    g.cache4_append(h, 700, we.F16, g.buffer(ka), g.buffer(va), ints(g, [0]), lens)
    c = C.Cache(1, 8, 64, 704)
    c.put(0, 0, k[0], v[0])
    q, qa = rows(rng, 1, 1, 64, 64, dtype)
    o, w = g.buffer(qa.nbytes), g.buffer(8 * cap * 4)
    g.cache4_attention(h, 1, 64, True, dtype, g.buffer(qa), lens, o, weight_out=w)
    want, received, bounds = C.attention(c, q, [700], [1], True)
    got = C.value(g.read(o, dtype=C.NP[dtype]).reshape(q.shape), dtype)
    assert (np.abs(got - want) <= C.tolerance(want, bounds, dtype)).all()
    gw = g.read(w, dtype=np.float32).reshape(8, cap)
    assert (np.abs(gw[:, :700] - received[0, :, :700]) <= C.weight_tolerance(received, bounds)[0, :, :700] + gw[:, :700] * 2.0 ** -24).all()
    assert not gw[:, 700:].any()


def test_attention_pads_are_not_read(scope):
    """Queries behind a sequence's count may hold anything; a call without tokens still writes weights."""
    g, rng = scope, np.random.default_rng(17)
    c = filled(rng, 2, 2, 128, 128, [90, 70])
    q, qa = rows(rng, 2, 12, 4, 128, we.F16)
    qa = qa.reshape(2, 12, -1)
    qa[0, 5:], qa[1, 1:] = NAN_BITS[we.F16], NAN_BITS[we.F16]
    q[0, 5:], q[1, 1:] = 0, 0
    check_attention(g, c, q, qa, [90, 70], [5, 1], True, we.F16)
    w = g.buffer(np.full(2 * 2 * 128, 2, np.float32))
    g.cache4_attention(c.handle(g), 0, 4, True, we.F16, None, ints(g, [90, 70]), None, weight_out=w)
    got = g.read(w, dtype=np.float32).reshape(2, 2, 128)
    assert (got[0, :, :90] == 0).all() and (got[0, :, 90:] == 2).all() and (got[1, :, :70] == 0).all()


# ---------------------------------------------------------------------------------------------------------- evict

def evict_case(rng, batch, kv, cap, lens, kind):
    weight = np.exp(2 * rng.standard_normal((batch, kv, cap))).astype(np.float32)
    pos = np.zeros((batch, kv, cap), np.int32)
    for b, n in enumerate(lens):
        for h in range(kv):
            pos[b, h, :n] = rng.permutation(n)
    if kind == "ties":
        weight = np.floor(weight * 2).astype(np.float32) / 2
    elif kind == "zero":
        weight[:] = 0
    elif kind == "special":
        weight[rng.random(weight.shape) < 0.1] = np.nan
        weight[rng.random(weight.shape) < 0.2] = np.float32(-0.0)
        weight[rng.random(weight.shape) < 0.1] = -1.5
        weight[rng.random(weight.shape) < 0.05] = np.inf
        weight[rng.random(weight.shape) < 0.05] = 1e-42
    return weight, pos


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,kv,dim,cap,lens,keep,sinks,recent,kind", [
    (1, 1, 64, 64, [1], 1, 0, 0, "plain"),                     # nothing to do
    (1, 1, 64, 64, [2], 1, 0, 0, "plain"),
    (2, 2, 128, 128, [100, 60], 99, 4, 10, "plain"),           # one slot of one sequence
    (2, 3, 192, 320, [300, 31], 64, 0, 0, "ties"),
    (2, 1, 64, 128, [104, 103], 100, 2, 5, "zero"),            # four and three slots, found one by one, all of one weight
    (2, 1, 128, 128, [105, 101], 100, 0, 0, "special"),        # five slots and one
    (1, 2, 128, 2112, [2104], 2100, 3, 2099, "special"),       # four, most of them protected
    (1, 2, 256, 256, [256], 0, 0, 0, "plain"),                 # all of them
    (1, 2, 128, 256, [250], 100, 40, 80, "plain"),             # nearly all protected
    (1, 2, 128, 256, [250], 100, 60, 150, "plain"),            # more protected than may stay
    (2, 1, 128, 192, [190, 0], 90, 0, 0, "zero"),              # one key: the lowest slots go
    (3, 2, 64, 1088, [1080, 1024, 500], 400, 2, 33, "special"),
    (1, 2, 64, 20480, [20001], 7000, 4, 512, "plain"),
    (1, 1, 64, 70016, [70001], 70000, 4, 512, "ties"),
])
def test_evict(scope, in_place, batch, kv, dim, cap, lens, keep, sinks, recent, kind):
    g, rng = scope, np.random.default_rng(cap + keep)
    c = C.Cache(batch, kv, dim, cap, fill=rng)
    h = c.handle(g)
    weight, pos = evict_case(rng, batch, kv, cap, lens, kind)
    seen = [n + 3 for n in lens]
    bufs = [ints(g, lens), g.buffer(weight), g.buffer(pos)]
    outs = bufs if in_place else [ints(g, [-1] * batch), g.buffer(np.full_like(weight, 5)), g.buffer(np.full_like(pos, 5))]
    g.cache4_evict(h, keep, bufs[0], outs[0], bufs[1], outs[1], bufs[2], outs[2], ints(g, seen), sinks, recent)
    left, w, p = C.evict(c, keep, lens, weight, pos, seen, sinks, recent)
    assert g.read(outs[0], dtype=np.int32).tolist() == left
    gw, gp = (g.read(o, dtype=np.uint32).reshape(weight.shape) for o in outs[1:])
    for b, n in enumerate(left):
        assert np.array_equal(gp[b, :, :n], p.view(np.uint32)[b, :, :n])
        assert np.array_equal(gw[b, :, :n], w.view(np.uint32)[b, :, :n])
        if not in_place:
            assert (gp[b, :, n:] == 5).all() and (gw[b, :, n:] == np.float32(5).view(np.uint32)).all()
    assert np.array_equal(g.read(h.data), c.bytes)


def test_evict_max_len_and_default_seen(scope):
    g, rng = scope, np.random.default_rng(2)
    c = C.Cache(2, 1, 64, 256, fill=rng)
    h = c.handle(g)
    weight, pos = evict_case(rng, 2, 1, 256, [200, 150], "plain")
    lens, out = ints(g, [200, 150]), ints(g, [0, 0])
    wo, po = g.buffer(weight.nbytes), g.buffer(pos.nbytes)
    g.cache4_evict(h, 50, lens, out, g.buffer(weight), wo, g.buffer(pos), po, recent=20, max_len=160)
    left, w, p = C.evict(c, 50, [160, 150], weight, pos, [200, 150], 0, 20)
    assert g.read(out, dtype=np.int32).tolist() == left == [50, 50]
    assert np.array_equal(g.read(po, dtype=np.int32).reshape(pos.shape)[:, :, :50], p[:, :, :50])
    assert np.array_equal(g.read(h.data), c.bytes)


# -------------------------------------------------------------------------------------------------------- together

class Decoder:
    """A decoding program and, beside it, the plain form's state."""

    def __init__(self, graph, seed, batch=2, heads=6, kv=2, dim=128, cap=256):
        self.g, self.rng, self.heads = graph, np.random.default_rng(seed), heads
        self.cache = we.Cache4(graph, batch, kv, dim, cap)
        self.c = C.Cache(batch, kv, dim, cap)
        self.lens, self.seen = [0] * batch, [0] * batch
        self.pos, self.weight = np.zeros((batch, kv, cap), np.int32), np.zeros((batch, kv, cap))

    def rows(self, tokens):
        return tuple(rows(self.rng, self.c.batch, tokens, h, self.c.dim, we.BF16) for h in (self.heads, self.c.kv, self.c.kv))

    def plain(self, data, tokens, counts, keep, sinks, recent):
        (q, _), (k, _), (v, _) = data
        for b, n in enumerate(counts):
            at = self.lens[b]
            self.c.put(b, at, k[b, :n], v[b, :n])
            self.pos[b, :, at:at + n] = self.seen[b] + np.arange(n)
            self.weight[b, :, at:at + n] = 0
            self.lens[b] += n
            self.seen[b] += n
        out, received, bounds = C.attention(self.c, q, self.lens, counts, True)
        self.weight += received
        return out, bounds

    def evict_from(self, weight, keep, sinks, recent):
        """the plain eviction, by the weights the GPU holds (an order of nearly equal sums is the sums')"""
        self.lens, self.weight, self.pos = C.evict(self.c, keep, self.lens, weight, self.pos, self.seen, sinks, recent)
        self.weight = self.weight.astype(np.float64)


def test_prompt_then_decoding_with_evictions(scope):
    """A padded prompt, then decode steps that keep the cache at its budget: each step's outputs, weights, positions and
    lengths against the plain form's, whose evictions go by the weights that the GPU accumulated."""
    g, d = scope, Decoder(scope, 20)
    keep, sinks, recent = 70, 2, 16
    steps = [(90, [90, 61])] + [(1, [1, 1])] * 6 + [(3, [3, 2])]
    for tokens, counts in steps:
        data = d.rows(tokens)
        out, bounds = d.plain(data, tokens, counts, keep, sinks, recent)
        qb, kb, vb = (g.buffer(a) for _, a in data)
        cb = ints(g, counts)
        d.cache.append(kb, vb, tokens, we.BF16, counts=cb)
        y = d.cache.attention(qb, tokens, d.heads, we.BF16, counts=cb, track=True)
        got = C.value(g.read(y, dtype=np.uint16).reshape(out.shape), we.BF16)
        live = ~np.isnan(out)
        assert (np.abs(got - out)[live] <= C.tolerance(out, bounds, we.BF16)[live]).all()
        w = g.read(d.cache.weight, dtype=np.float32).reshape(d.weight.shape)
        for b, n in enumerate(d.lens):
            tol = C.weight_tolerance(d.weight, bounds)[b, :, :n] * 2 + 1e-6
            assert (np.abs(w[b, :, :n] - d.weight[b, :, :n]) <= tol).all()
        d.cache.evict(keep, sinks, recent)
        d.evict_from(w, keep, sinks, recent)
        assert g.read(d.cache.lens, dtype=np.int32).tolist() == d.lens
        assert g.read(d.cache.seen, dtype=np.int32).tolist() == d.seen
        p = g.read(d.cache.pos, dtype=np.int32).reshape(d.pos.shape)
        for b, n in enumerate(d.lens):
            assert np.array_equal(p[b, :, :n], d.pos[b, :, :n])
            assert {*p[b, 0, :n]} >= {0, 1}  # the first tokens stay
    d.cache.free()


@pytest.mark.parametrize("stream", [0, 1])
def test_captured_decode_step_replays(scope, stream):
    """One captured step (append, attention with weights, evict) replayed as its lengths grow, beside an eager twin. Each
    replay's outputs and state equal the eager call's bit for bit; two graphs share the stream's scratch."""
    g = scope
    batch, heads, kv, dim, cap, keep = 2, 8, 2, 128, 2048, 1500
    rng = np.random.default_rng(30 + stream)
    k0, ka = rows(rng, batch, 1490, kv, dim, we.F16)
    _, va = rows(rng, batch, 1490, kv, dim, we.F16)
    g.sync()
    g.stream(stream)
    try:
        twins = []
        for _ in range(2):
            c = we.Cache4(g, batch, kv, dim, cap)
            c.append(g.buffer(ka), g.buffer(va), 1490, we.F16)
            twins.append(c)
        bufs = [g.buffer(batch * h * dim * 2) for h in (heads, kv, kv)]
        outs = [g.buffer(batch * heads * dim * 2) for _ in twins]

        def step(c, out):
            c.append(bufs[1], bufs[2], 1, we.F16)
            g.cache4_attention(c, 1, heads, True, we.F16, bufs[0], c.lens, out, weight=c.weight, weight_out=c.weight)
            c.evict(keep, 4, 64)

        def fresh():
            for b, h in zip(bufs, (heads, kv, kv)):
                g.write(b, rows(rng, batch, 1, h, dim, we.F16)[1])

        fresh()
        for c, o in zip(twins, outs):  # an eager step of each first
            step(c, o)
        g.sync()
        graphs = []
        for _ in range(2):
            g.graph_begin()
            step(twins[0], outs[0])
            graphs.append(g.graph_end())
        try:
            for rep in range(14):  # past the budget: the last ones evict
                fresh()
                g.graph_launch(graphs[rep % 2])
                step(twins[1], outs[1])
                assert np.array_equal(g.read(outs[0]), g.read(outs[1])), rep
            for name in ("lens", "seen", "pos", "weight", "data"):
                assert np.array_equal(g.read(getattr(twins[0], name)), g.read(getattr(twins[1], name))), name
            assert g.read(twins[0].lens, dtype=np.int32).tolist() == [keep] * batch
        finally:
            g.sync()
            for x in graphs:
                g.graph_destroy(x)
    finally:
        g.stream(0)
        g.fork()
        g.join()


def test_rows_of_a_fused_projection(scope):
    """q, k and v as columns of one QKV row, read by stride, with the projection's own norm and rotation before: the same
    bytes as from packed copies."""
    g, rng = scope, np.random.default_rng(41)
    batch, heads, kv, d, hidden = 3, 4, 2, 128, 256
    n = (heads + 2 * kv) * d
    x = g.buffer(C.store(rng.standard_normal((batch, hidden)), we.BF16))
    w = g.buffer(C.store(rng.standard_normal((n, hidden)) / 16, we.BF16))
    ones, angle = g.buffer(np.zeros(d, np.float32)), rng.uniform(0, 6, (batch, d // 2)).astype(np.float32)
    qkv = g.buffer(batch * n * 2)
    g.matmul_qk_norm_rope(we.matmul_params(batch, n, hidden, 1.0, graph=g), we.BF16, x, we.BF16, w, we.BF16, qkv, heads, kv, 1e-6,
                          1.0, ones, ones, 0, g.buffer(np.cos(angle)), g.buffer(np.sin(angle)))
    a = g.read(qkv, dtype=np.uint16).reshape(batch, n)
    parts = [g.buffer(np.ascontiguousarray(p)) for p in np.split(a, [heads * d, (heads + kv) * d], 1)]
    got = []
    for q, k, v, st in ((qkv, qkv.ptr + heads * d * 2, qkv.ptr + (heads + kv) * d * 2, n), (*parts, 0)):
        c = we.Cache4(g, batch, kv, d, 64)
        for _ in range(2):
            c.append(k, v, 1, we.BF16, k_stride=st, v_stride=st)
        y = c.attention(q, 1, heads, we.BF16, q_stride=st, track=True)
        got.append([g.read(b) for b in (y, c.data, c.weight)])
    assert all(np.array_equal(p, q) for p, q in zip(*got)) and got[0][0].any()


def test_two_streams_at_once(scope):
    """Calls on both compute streams, each with its own scratch, queued without a wait between them."""
    g, rng = scope, np.random.default_rng(40)
    c = filled(rng, 2, 2, 128, 4096, [4001, 3000])
    q, qa = rows(rng, 2, 1, 8, 128, we.BF16)
    h, lens, qb = c.handle(g), ints(g, [4001, 3000]), g.buffer(qa)
    outs = [(g.buffer(qa.nbytes), g.buffer(2 * 2 * 4096 * 4)) for _ in range(4)]
    g.sync()
    g.fork()
    for i, (o, w) in enumerate(outs):
        g.stream(i % 2)
        g.cache4_attention(h, 1, 8, True, we.BF16, qb, lens, o, weight_out=w)
    g.stream(0)
    g.join()
    got = [(g.read(o), g.read(w)) for o, w in outs]
    assert all(np.array_equal(a, b) for x in got[1:] for a, b in zip(x, got[0]))


# -------------------------------------------------------------------------------------------------------- refusals

def test_refusals(scope):
    g = scope
    c = we.Cache4(g, 2, 2, 128, 64)
    q, out, kv = g.buffer(2 * 8 * 128 * 2), g.buffer(2 * 8 * 128 * 2), g.buffer(2 * 2 * 128 * 2)
    small, wide = g.buffer(4), g.buffer(2 * 2 * 64 * 4)
    bf = we.BF16

    def refused(match, call, *a, code=we.WE_EINVAL, **kw):
        with pytest.raises(we.WeError, match=match) as e:
            call(*a, **kw)
        assert e.value.code == code

    for bad, match, code in (((2, 2, 96, 64), "dim must be a multiple of 64", 4), ((2, 2, 320, 64), "at most 256, got 320", 4),
                             ((2, 2, 128, 100), "capacity must be a multiple of 64", 1),
                             ((0, 2, 128, 64), "batch and kvHeads must be from 1", 1),
                             ((2, 0, 128, 64), "batch and kvHeads must be from 1", 1)):
        refused(match, we.Cache4, g, *bad, code=code)
    refused("cache data is too small", g.cache4_load, we.Cache4(g, 2, 2, 128, 64, data=small), 1, bf, kv, None, lens=c.lens)
    refused("cache data must be 16-byte aligned", g.cache4_load, we.Cache4(g, 2, 2, 128, 64, data=c.data.ptr + 4), 1, bf, kv,
            None, lens=c.lens)
    for bad, match in (((1, we.FP8, kv, kv), "dtype 3 is not"), ((1, bf, None, kv), "k or v is null"),
                       ((2, bf, kv, kv), "k is too small")):
        refused(match, g.cache4_append, c, *bad, c.lens, c.lens)
    refused("stride below", g.cache4_append, c, 1, bf, kv, kv, c.lens, c.lens, k_stride=128)
    refused("stride must be a multiple of 8", g.cache4_append, c, 1, bf, kv, kv, c.lens, c.lens, v_stride=260)
    refused("k must be 16-byte aligned", g.cache4_append, c, 1, bf, kv.ptr + 2, kv, c.lens, c.lens)
    refused("lens or lens_out is null", g.cache4_append, c, 1, bf, kv, kv, c.lens, None)
    refused("lens_out is too small", g.cache4_append, c, 1, bf, kv, kv, c.lens, small)
    refused("seen_out without seen", g.cache4_append, c, 1, bf, kv, kv, c.lens, c.lens, seen_out=c.seen)
    refused("seen_out overlaps lens", g.cache4_append, c, 1, bf, kv, kv, c.lens, g.buffer(8), seen=c.seen, seen_out=c.lens)
    refused("pos overlaps|weight overlaps", g.cache4_append, c, 1, bf, kv, kv, c.lens, c.lens, pos=wide, weight=wide)
    refused("cache data overlaps k", g.cache4_append, c, 1, bf, c.data, kv, c.lens, c.lens)

    def attention(tokens=1, heads=8, dtype=bf, q=q, lens=c.lens, out=out, cache=c, **kw):
        g.cache4_attention(cache, tokens, heads, True, dtype, q, lens, out, **kw)

    refused("heads must be a multiple of kvHeads", attention, heads=3)
    refused("heads must be a multiple of kvHeads", attention, heads=0)
    refused("dtype 4 is not", attention, dtype=we.INT4)
    refused("lens is null", attention, lens=None)
    refused("q or out is null", attention, q=None)
    refused("(q|out) is too small", attention, tokens=2)
    refused("out overlaps q", attention, out=q)
    refused("weight without weight_out", attention, weight=c.weight)
    refused("weight_out is too small", attention, weight_out=small)
    refused("weight_out overlaps cache data", attention, weight_out=c.data)
    refused("out stride must be", attention, out_stride=1028)
    refused("at most 16777216 tokens", attention, tokens=(1 << 24) + 1)
    freed = g.buffer(64)
    g.free(freed)
    args = (c, 4, c.lens, c.lens, c.weight, c.weight, c.pos, c.pos)
    refused("needs lens, weight and pos", g.cache4_evict, c, 4, c.lens, c.lens, None, c.weight, c.pos, c.pos)
    refused("cache data overlaps pos_out", g.cache4_evict, c, 4, c.lens, c.lens, c.weight, c.weight, c.pos, c.data)
    refused("weight_out overlaps pos", g.cache4_evict, c, 4, c.lens, c.lens, c.weight, c.pos, c.pos, wide)
    refused("below 2\\^31", g.cache4_evict, *args, sinks=1 << 31)
    refused("lens is too small", g.cache4_evict, c, 4, small, c.lens, c.weight, c.weight, c.pos, c.pos)
    refused("heads must be a multiple", c.attention, q, 1, 3, bf)
    # and the calls as they should be
    g.cache4_append(c, 1, bf, kv, kv, c.lens, c.lens)
    attention()
    g.cache4_evict(*args)
    assert g.read(c.lens, dtype=np.int32).tolist() == [1, 1]


def test_a_capture_needs_its_scratch(scope):
    """A call whose scratch the context does not hold yet is refused inside a capture, and the capture goes on."""
    fresh = we.Graph(0)
    try:
        c = we.Cache4(fresh, 1, 1, 64, 64)
        buf = fresh.buffer(64 * 2)
        out, wo = fresh.buffer(64 * 2), fresh.buffer(64 * 4)
        fresh.graph_begin()
        with pytest.raises(we.WeError, match="run the call once before capturing it"):
            fresh.cache4_attention(c, 1, 1, True, we.F16, buf, c.lens, out, weight_out=wo)
        fresh.graph_destroy(fresh.graph_end())
        fresh.cache4_attention(c, 1, 1, True, we.F16, buf, c.lens, out, weight_out=wo)
        assert not fresh.read(out).any()
    finally:
        fresh.destroy()
