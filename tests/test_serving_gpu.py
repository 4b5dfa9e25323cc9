"""Serving operators of a ragged batch on the GPU against their plain 64-bit forms: rotating cache append, chunk attention over
the paged cache, token sampling; caller-owned memory, captured graphs, and a run of the operators together."""
import ctypes as C

import numpy as np
import pytest

from fandhe_ai_b200 import BF16, F32, Backend, BackendError
from fandhe_ai_b200 import paged_kv as P
from fandhe_ai_b200.decoder import SampleArgs, sample_tokens
from oracle import oracle as O

from serving_ref import Batch, append_ref, attention_ref, bf16, sample_ref

pytestmark = pytest.mark.gpu


def up(be, x, as_bf16=False):
    return be.upload(O.f32_to_bf16(np.ascontiguousarray(x, np.float32)) if as_bf16 else np.ascontiguousarray(x))


def down(buf, shape, as_bf16=False):
    x = buf.numpy()
    return (O.bf16_to_f32(x.view(np.uint16)) if as_bf16 else x.view(np.float32)).reshape(shape)


def index_buffers(be, bt):
    return be.upload(bt.tables), be.upload(bt.q_starts), be.upload(bt.seq_lens)


def layout_of(bt):
    return P.PagedKvLayout(bt.blocks, bt.block, bt.kv_heads * bt.dh, BF16 if bt.pool_bf16 else F32)


# ------------------------------------------------------------------------------------------ append

APPEND = [
    dict(new=[1], total=[1]),
    dict(new=[1, 1, 1], total=[5, 17, 32]),
    dict(new=[3, 0, 40, 1], total=[3, 9, 57, 16], pad_rows=3),
    dict(new=[7, 130], total=[300, 130], heads=12, kv_heads=12, dh=64),
    dict(new=[5, 2], total=[5, 33], heads=6, kv_heads=2, dh=80, block=8),
    dict(new=[5, 2], total=[5, 33], heads=3, kv_heads=1, dh=10, block=1),
    dict(new=[4, 4], total=[260, 4], heads=4, kv_heads=4, dh=256, block=256, pool_bf16=False),
    dict(new=[2] * 300, total=[4] * 300, heads=2, kv_heads=1, dh=64),          # more sequences than a block has threads
]


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("case", APPEND)
def test_append_matches_the_plain_form(be, case, adjacent, io_bf16):
    bt = Batch(seed=3, **case)
    for rotary in sorted({bt.dh // 2 // 2 * 2, bt.dh, 0}):
        width = (bt.heads + 2 * bt.kv_heads) * bt.dh
        stride = width + (2 if rotary == bt.dh else 0)             # rows further apart than they are long
        rng = np.random.default_rng(4)
        qkv = rng.standard_normal((bt.rows, stride)).astype(np.float32)
        if io_bf16:
            qkv = bf16(qkv)
        n_pos = max(bt.total) + 1
        cos, sin = P.rope_table(10000.0, max(2, rotary), n_pos)
        tables, starts, lens = index_buffers(be, bt)
        kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
        q0 = np.full((bt.rows, bt.heads * bt.dh), 77.0, np.float32)
        q = up(be, q0, io_bf16)
        args = P.RopeAppendArgs(layout_of(bt), bt.batch, bt.rows, bt.heads, bt.kv_heads, bt.width, rotary, n_pos, adjacent,
                                BF16 if io_bf16 else F32, stride)
        P.rope_paged_kv_append(be, up(be, qkv, io_bf16), be.upload(cos), be.upload(sin), tables, starts, lens, kp, vp, args, q)
        (rq, rk, rv), (mq, mk, mv) = append_ref(bt, qkv[:, :width], cos, sin, rotary, adjacent)
        live = ~np.isnan(rq[:, 0])
        got = down(q, q0.shape, io_bf16)
        step = 2.0 ** -8 if io_bf16 else 0.0
        assert (np.abs(got[live] - rq[live]) <= mq[live] * 2.0 ** -23 + step * np.abs(rq[live]) * 1.001).all()
        assert (got[~live] == 77.0).all()                          # rows behind the last sequence
        step = 2.0 ** -8 if bt.pool_bf16 else 0.0
        k = down(kp, bt.k.shape, bt.pool_bf16)
        assert (np.abs(k - rk) <= mk * 2.0 ** -23 + step * np.abs(rk) * (mk > 0) * 1.001).all()
        want_v = bf16(rv) if bt.pool_bf16 else rv.astype(np.float32)
        assert np.array_equal(down(vp, bt.v.shape, bt.pool_bf16), want_v.reshape(bt.v.shape))


def test_append_without_rotation_needs_no_table(be):
    bt = Batch([3, 2], [20, 2], heads=4, kv_heads=1, dh=64, seed=5)
    qkv = np.random.default_rng(6).standard_normal((5, 6 * 64)).astype(np.float32)
    tables, starts, lens = index_buffers(be, bt)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    q, none = be.alloc_zeroed((5, 256)), be.alloc_zeroed((0,))
    args = P.RopeAppendArgs(layout_of(bt), 2, 5, 4, 1, bt.width, 0, 0)
    P.rope_paged_kv_append(be, be.upload(qkv), none, none, tables, starts, lens, kp, vp, args, q)
    assert np.array_equal(q.numpy(), qkv[:, :256])


def test_rows_before_the_first_sequence_are_left_alone(be):
    """q_starts that begin above zero are outside the contract; the rows before them still are not touched."""
    bt = Batch([3, 2], [20, 2], heads=4, kv_heads=1, dh=64, seed=5, pad_rows=4)
    bt.q_starts = (bt.q_starts + 4).astype(np.uint32)
    tables, starts, lens = index_buffers(be, bt)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    qkv = be.upload(np.ones((9, 6 * 64), np.float32))
    cos, sin = P.rope_table(10000.0, 64, 32)
    q = be.upload(np.full((9, 256), 7.0, np.float32))
    args = P.RopeAppendArgs(layout_of(bt), 2, 9, 4, 1, bt.width, 64, 32)
    P.rope_paged_kv_append(be, qkv, be.upload(cos), be.upload(sin), tables, starts, lens, kp, vp, args, q)
    assert (q.numpy()[:4] == 7.0).all() and (q.numpy()[4:] != 7.0).any()
    for seqs in (1, 2):                    # one launch, and with the keys shared out and joined
        long = Batch([3], [4000], heads=4, kv_heads=1, dh=64 * seqs, seed=5, pad_rows=4)
        long.q_starts = (long.q_starts + 4).astype(np.uint32)
        t2, s2, l2 = index_buffers(be, long)
        out = be.upload(np.full((7, 4 * long.dh), 7.0, np.float32))
        ca = P.PagedChunkArgs(layout_of(long), 1, 7, 3, 4000, 4, 1, long.width, 0.1)
        ws = be.alloc_zeroed((max(16, P.paged_chunk_workspace(be, ca)),), np.uint8)
        P.paged_chunk_attention(be, be.upload(long.q), be.upload(long.pool_array(long.k)), be.upload(long.pool_array(long.v)), t2, s2, l2, ca, ws, out)
        assert (out.numpy()[:4] == 7.0).all() and (out.numpy()[4:] != 7.0).any()


def test_append_with_positions_of_its_own(be):
    bt = Batch([3, 2], [20, 2], heads=4, kv_heads=1, dh=64, seed=5)
    qkv = np.random.default_rng(6).standard_normal((5, 6 * 64)).astype(np.float32)
    pos = np.array([100, 7, 0, 511, 3], np.uint32)
    cos, sin = P.rope_table(500000.0, 64, 512)
    tables, starts, lens = index_buffers(be, bt)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    q = be.alloc_zeroed((5, 256))
    args = P.RopeAppendArgs(layout_of(bt), 2, 5, 4, 1, bt.width, 64, 512)
    P.rope_paged_kv_append(be, be.upload(qkv), be.upload(cos), be.upload(sin), tables, starts, lens, kp, vp, args, q, be.upload(pos))
    (rq, rk, _), (mq, mk, _) = append_ref(bt, qkv, cos, sin, 64, False, pos)
    assert (np.abs(q.numpy() - rq) <= mq * 2.0 ** -23).all()
    assert (np.abs(down(kp, bt.k.shape, True) - rk) <= mk * 2.0 ** -23 + 2.0 ** -8 * np.abs(rk) * (mk > 0) * 1.001).all()


# ------------------------------------------------------------------------------------------ attention

def run_attention(be, bt, q, io_bf16, scale, stride=0, max_q=None, max_len=None, workspace=None, fill=55.0):
    tables, starts, lens = index_buffers(be, bt)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    width = bt.heads * bt.dh
    buf = np.zeros((bt.rows, stride or width), np.float32)
    buf[:, :width] = q
    args = P.PagedChunkArgs(layout_of(bt), bt.batch, bt.rows, max_q if max_q is not None else max(bt.new),
                            max_len if max_len is not None else max(bt.total), bt.heads, bt.kv_heads, bt.width, scale,
                            BF16 if io_bf16 else F32, stride)
    P.validate_ragged_batch(bt.tables, bt.q_starts, bt.seq_lens, args)
    need = P.paged_chunk_workspace(be, args)
    ws = workspace or be.upload(np.full(max(1, need), 0xFF, np.uint8))         # whatever stands in it must not matter
    out = up(be, np.full((bt.rows, width), fill, np.float32), io_bf16)
    P.paged_chunk_attention(be, up(be, buf, io_bf16), kp, vp, tables, starts, lens, args, ws, out)
    return down(out, (bt.rows, width), io_bf16)


def check_attention(be, bt, io_bf16, scale=None, **kw):
    scale = bt.dh ** -0.5 if scale is None else scale
    q = bf16(bt.q) if io_bf16 else bt.q
    got = run_attention(be, bt, q, io_bf16, scale, **kw)
    ref, bound = attention_ref(bt, q, scale, split_terms=not io_bf16)
    live = ~np.isnan(ref[:, 0])
    assert (got[~live] == 55.0).all(), "rows behind the last sequence were written"
    err = np.abs(got[live] - ref[live])
    step = 2.0 ** -8 if io_bf16 else 2.0 ** -24
    lim = bound[live] + step * 1.001 * (np.abs(ref[live]) + bound[live])
    worst = np.unravel_index(np.argmax(err - lim), err.shape)
    assert (err <= lim).all(), f"worst at {worst}: off by {err[worst]:.3g}, allowed {lim[worst]:.3g}"


ATTENTION = [
    dict(new=[1], total=[1]),
    dict(new=[1], total=[16]),
    dict(new=[1, 1, 1, 1], total=[2, 127, 128, 129]),
    dict(new=[2], total=[2]),
    dict(new=[4, 4], total=[1000, 260]),
    dict(new=[33], total=[33]),
    dict(new=[3, 0, 0, 65], total=[3, 40, 0, 300], pad_rows=5),
    dict(new=[129, 1], total=[129, 513]),
    dict(new=[257], total=[400], heads=4, kv_heads=4),
    dict(new=[64, 1, 17], total=[64, 777, 190], heads=2, kv_heads=2, dh=64),
    dict(new=[50, 5], total=[170, 600], heads=12, kv_heads=4, dh=64),          # three query heads to a KV head
    dict(new=[20, 40], total=[20, 333], heads=8, kv_heads=1),
    dict(new=[20, 40], total=[20, 333], heads=20, kv_heads=1, dh=64),
    dict(new=[9, 30], total=[70, 30], block=8),
    dict(new=[9, 130], total=[70, 300], block=32),
    dict(new=[9, 30], total=[300, 30], block=64, dh=64, heads=4, kv_heads=2),
    dict(new=[9, 30], total=[300, 30], block=256, heads=4, kv_heads=2),
    dict(new=[9, 3], total=[70, 5], block=1),                                   # the general kernel from here on
    dict(new=[9, 3], total=[70, 50], dh=80),
    dict(new=[9, 3], total=[70, 50], dh=256, heads=2, kv_heads=1),
    dict(new=[9, 3], total=[70, 50], heads=4, kv_heads=4, pool_bf16=False),
    dict(new=[1] * 150, total=list(range(1, 151)), heads=4, kv_heads=2, dh=64),
]


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", ATTENTION)
def test_attention_matches_the_plain_form(be, case, io_bf16):
    check_attention(be, Batch(seed=7, **case), io_bf16)


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_ignores_what_no_token_sees(be, dh, io_bf16):
    """NaN and infinities in unused blocks and behind every sequence's end, in K and in V."""
    check_attention(be, Batch([5, 1, 70], [37, 200, 70], dh=dh, seed=8, poison=True), io_bf16)


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_attention_non_finite_values_reach_only_the_tokens_that_see_them(be, value, io_bf16):
    """A non-finite value at a new token's place: earlier tokens must not notice, later ones must."""
    bt = Batch([40, 3], [140, 300], heads=4, kv_heads=2, seed=9)
    blk, off = bt.places(0)
    at = 120                                                        # new token 20 of sequence 0
    bt.v[blk[at], off[at], 5] = value                               # head 0, element 5
    q = bf16(bt.q) if io_bf16 else bt.q
    got = run_attention(be, bt, q, io_bf16, 0.1)
    clean = Batch([40, 3], [140, 300], heads=4, kv_heads=2, seed=9)
    ref, bound = attention_ref(clean, q, 0.1, split_terms=not io_bf16)
    touched = np.zeros(got.shape, bool)
    for h in (0, 1):                                                # the query heads of KV head 0
        touched[20:40, h * 128 + 5] = True
    step = 2.0 ** -8 if io_bf16 else 2.0 ** -24
    assert (np.abs(got - ref) <= bound + step * 1.001 * (np.abs(ref) + bound))[~touched].all()
    assert (np.isnan(got[touched]) if np.isnan(value) else got[touched] == value).all()


@pytest.mark.parametrize("io_bf16", [False, True])
def test_attention_large_and_tiny_scores(be, io_bf16):
    """Scores of hundreds (one key wins), a scale of zero (all keys alike) and a negative scale."""
    bt = Batch([30, 1], [200, 300], heads=4, kv_heads=2, seed=10, q_scale=20.0)
    for scale in (0.3, 0.0, -0.05):
        check_attention(be, bt, io_bf16, scale=scale)


@pytest.mark.parametrize("io_bf16", [False, True])
def test_attention_strided_queries_and_loose_bounds(be, io_bf16):
    """Queries inside wider rows; max_q_len and max_seq_len far above what the batch holds."""
    bt = Batch([11, 2], [90, 44], heads=6, kv_heads=2, dh=64, seed=11)
    bt.width, bt.tables = 40, np.pad(bt.tables, ((0, 0), (0, 40 - bt.width)), constant_values=P.SENTINEL)
    check_attention(be, bt, io_bf16, stride=6 * 64 + 24, max_q=500, max_len=640)


def test_attention_long_cache_split_over_blocks(be):
    """Few rows over a long cache: the keys of a row are shared out and joined."""
    check_attention(be, Batch([2, 1], [9000, 5001], heads=4, kv_heads=1, seed=12), False)
    check_attention(be, Batch([2, 1], [9000, 5001], heads=4, kv_heads=1, seed=12), True)
    check_attention(be, Batch([3], [4100], heads=2, kv_heads=2, dh=64, seed=13), False)


def test_attention_twice_on_one_workspace_is_the_same(be):
    bt = Batch([64, 1, 17], [900, 777, 190], seed=14)
    q = bf16(bt.q)
    ws = be.upload(np.full(1 << 26, 0xAB, np.uint8))
    a = run_attention(be, bt, q, True, 0.1, workspace=ws)
    b = run_attention(be, bt, q, True, 0.1, workspace=ws)
    assert np.array_equal(a, b)
    small = Batch([1], [3000], seed=15)                              # another shape on the same workspace, then the first again
    check_attention(be, small, True, workspace=ws)
    assert np.array_equal(a, run_attention(be, bt, q, True, 0.1, workspace=ws))


@pytest.mark.parametrize("kind", ["block", "long", "rows", "planned rows"])
@pytest.mark.parametrize("dh", [64, 80])
def test_attention_bad_device_arrays_are_reported(kind, dh):
    """What only the device sees: reported by the next synchronisation; the other sequence is still right."""
    be = Backend(0)
    try:
        bt = Batch([4, 4], [100, 60], heads=4, kv_heads=2, dh=dh, seed=16)
        good = attention_ref(bt, bt.q, 0.1)
        tables, lens, starts = bt.tables.copy(), bt.seq_lens.copy(), bt.q_starts.copy()
        if kind == "block":
            tables[0, 2] = bt.blocks + 5
        elif kind == "long":
            lens[0] = 101 + 16                                       # beyond max_seq_len
        elif kind == "rows":
            lens[0] = 3
        kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
        args = P.PagedChunkArgs(layout_of(bt), 2, 8, 3 if kind == "planned rows" else 4, 100, 4, 2, bt.width, 0.1)
        out = be.alloc_zeroed((8, 4 * dh))
        ws = be.alloc_zeroed((max(1, P.paged_chunk_workspace(be, args)),), np.uint8)
        P.paged_chunk_attention(be, be.upload(bt.q), kp, vp, be.upload(tables), be.upload(starts), be.upload(lens), args, ws, out)
        host = np.empty((8, 4 * dh), np.float32)
        st = P.lib().b200_download(be._ctx, out.handle, 0, host.ctypes.data_as(C.c_void_p), host.nbytes)
        assert st != 0 and "0x20" in P.lib().b200_last_error().decode()
        if kind != "planned rows":
            assert (np.abs(host[4:] - good[0][4:]) <= good[1][4:] + 2.0 ** -23 * np.abs(good[0][4:])).all()
        assert be.poisoned
    finally:
        be.close()


def test_refusals_that_need_a_context(be):
    bt = Batch([4, 4], [100, 60], heads=4, kv_heads=2, seed=16)
    tables, starts, lens = index_buffers(be, bt)
    pool = be.upload(bt.pool_array(bt.k))
    args = P.PagedChunkArgs(layout_of(bt), 2, 8, 4, 100, 4, 2, bt.width, 0.1)
    q, out = be.alloc_zeroed((8, 512)), be.alloc_zeroed((8, 512))
    ws = be.alloc_zeroed((max(16, P.paged_chunk_workspace(be, args)),), np.uint8)
    tiny = be.alloc_zeroed((4,))

    def refused(kind, **kw):
        d = dict(q=q, k_pool=pool, v_pool=pool, block_tables=tables, q_starts=starts, seq_lens=lens, args=args, workspace=ws, out=out)
        d.update(kw)
        with pytest.raises(BackendError) as e:
            P.paged_chunk_attention(be, **d)
        assert e.value.kind == kind

    for name in ("q", "k_pool", "v_pool", "block_tables", "q_starts", "seq_lens", "out"):
        refused("ShapeMismatch", **{name: tiny if name not in ("q_starts", "seq_lens") else be.alloc_zeroed((1,))})
    refused("InvalidArgument", q=be.alloc_zeroed((9, 512)), q_off=4)
    refused("InvalidArgument", out=be.alloc_zeroed((9, 512)), out_off=8)
    other = Backend(0)
    try:
        refused("DeviceMismatch", q=other.alloc_zeroed((8, 512)))
    finally:
        other.close()
    with pytest.raises(BackendError):
        sample_tokens(be, tiny, SampleArgs(1, 5), tiny, tiny)
    assert not be.poisoned


# ------------------------------------------------------------------------------------------ sampling

def draw(be, x, t=None, k=None, p=None, m=None, u=None, as_bf16=False, stride=0, with_extras=True):
    rows, vocab = x.shape
    full = np.full((rows, stride or vocab), 9e9, np.float32)          # what stands behind a row must not be looked at
    full[:, :vocab] = x
    buf = be.upload(np.ascontiguousarray(O.f32_to_bf16(full.ravel()) if as_bf16 else full))
    par = [None if a is None else be.upload(np.ascontiguousarray(np.broadcast_to(a, (rows,)), dtype=d)) for a, d in
           ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    ids = be.upload(np.full(rows, -7, np.int32))
    prob, kept = (be.alloc_zeroed((rows,)), be.alloc_zeroed((rows,), np.int32)) if with_extras else (None, None)
    sample_tokens(be, buf, SampleArgs(rows, vocab, stride, BF16 if as_bf16 else F32), be.upload(np.ascontiguousarray(u, np.float32)), ids, *par,
                  prob=prob, kept=kept)
    return ids.numpy(), prob.numpy() if prob else None, kept.numpy() if kept else None


def check_draw(be, x, t=1.0, k=0, p=1.0, m=0.0, u=None, seed=0, **kw):
    rows = x.shape[0]
    u = np.random.default_rng(seed).random(rows).astype(np.float32) if u is None else np.broadcast_to(np.float32(u), (rows,))
    x = bf16(x) if kw.get("as_bf16") else np.asarray(x, np.float32)
    t, k, p, m = (np.broadcast_to(np.asarray(a, d), (rows,)) for a, d in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32)))
    ids, prob, kept = draw(be, x, t, k, p, m, u, **kw)
    for r in range(rows):
        want = sample_ref(x[r], float(t[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]))
        assert want[3] > 1e-12 or want[3] == 0.0, "the row's borders are too close to decide in 64 bits: choose another seed"
        assert (ids[r], kept[r]) == (want[0], want[2]), f"row {r}: {ids[r], kept[r]} instead of {want}"
        assert abs(prob[r] - want[1]) <= 2.0 ** -23 * want[1]


@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 1000, 4097, 16384, 16385, 33333, 128256])
@pytest.mark.parametrize("as_bf16", [False, True])
def test_sampling_matches_the_plain_form(be, vocab, as_bf16):
    rng = np.random.default_rng(vocab)
    rows = 12 if vocab < 50000 else 6
    x = rng.standard_normal((rows, vocab)) * 2.5
    x[: rows // 2, rng.integers(0, vocab, 5)] += 6
    t = np.array([0.7, 1.0, 1.3, 0.05, 3.0, 0.0] * 2)[:rows]
    k = np.array([0, 50, 1, vocab, vocab + 5, 700] * 2)[:rows]
    p = np.array([0.9, 1.0, 0.5, 0.95, 0.3, 0.8, 0.999, 0.2, 1.0, 0.0, 0.6, 2.0])[:rows]
    m = np.array([0.0, 0.05, 0.0, 0.0, 0.3, 0.0, 0.1, 0.0, 0.0, 0.5, 1.0, 0.0])[:rows]
    check_draw(be, x, t, k, p, m, seed=vocab + 1, as_bf16=as_bf16)


@pytest.mark.parametrize("rows", [1, 3, 75, 300])
def test_sampling_row_counts_and_strides(be, rows):
    x = np.random.default_rng(rows).standard_normal((rows, 501)) * 3
    check_draw(be, x, 0.8, 40, 0.9, 0.01, seed=rows, stride=509)
    check_draw(be, x, 0.8, 40, 0.9, 0.01, seed=rows, stride=512, as_bf16=True)


def test_sampling_flat_and_tied_rows(be):
    """All logits equal, two values only, and a row in which one bin of the search holds thousands of tokens."""
    for vocab in (600, 20000):
        x = np.zeros((5, vocab), np.float32)
        x[1, ::2] = 1.0
        x[2] = np.random.default_rng(1).standard_normal(vocab) * 1e-4
        x[3] = -5.0
        x[4, 17] = 30.0
        for kw in (dict(k=vocab // 3), dict(p=0.37), dict(k=vocab // 2 + 1, p=0.61), dict(), dict(m=0.5), dict(t=1e30, p=0.5), dict(t=1e-30)):
            check_draw(be, x, u=np.float32(0.777), **kw)
            check_draw(be, x, u=np.float32(0.0), **kw)


def test_sampling_order_of_ties_and_borders(be):
    x = np.log(np.array([[4.0, 1.0, 4.0, 1.0]], np.float32))
    x[0, 1] = x[0, 3] = 0.0                                           # exactly e^(-ln 4) apart in f32 logits
    for u, kw, want in ((0.95, dict(k=3), 2), (0.95, dict(p=0.45), 2), (0.0, dict(), 0), (0.999, dict(), 3), (0.95, dict(k=1), 0)):
        ids, _, _ = draw(be, x, **{a: b for a, b in kw.items()}, u=[u])
        assert ids[0] == want
    # equal weights: sums are exact, a draw on a border goes to the token behind it
    ids, prob, kept = draw(be, np.zeros((4, 4), np.float32), u=[0.0, 0.25, 0.5, 0.75])
    assert ids.tolist() == [0, 1, 2, 3] and kept.tolist() == [4] * 4 and prob.tolist() == [0.25] * 4
    ids, _, kept = draw(be, np.zeros((1, 4), np.float32), p=0.5, u=[0.9])
    assert ids[0] == 1 and kept[0] == 2
    ids, _, kept = draw(be, np.array([[-0.0, 0.0, -0.0]], np.float32), k=2, u=[0.9])      # -0 and +0 are equal logits
    assert ids[0] == 1 and kept[0] == 2


def test_sampling_masked_rows_and_bad_parameters(be):
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((12, 3000)) * 2).astype(np.float32)
    x[0] = -np.inf
    x[1, :-1] = -np.inf
    x[2, 100] = np.nan
    x[3, 100] = np.inf
    x[4, rng.random(3000) < 0.95] = -np.inf
    x[5] = np.finfo(np.float32).min                                   # a mask of the type's lowest value leaves a flat row
    t = np.ones(12, np.float32)
    t[6], t[7], t[8] = -1.0, np.nan, np.inf
    u = rng.random(12).astype(np.float32)
    u[9], u[10] = 1.0, np.nan
    p = np.full(12, 0.9, np.float32)
    p[11] = np.nan
    ids, prob, kept = draw(be, x, t, None, p, None, u)
    for r in range(12):
        want = sample_ref(x[r], float(t[r]), 0, float(p[r]), 0.0, float(u[r]))
        assert (ids[r], kept[r]) == (want[0], want[2])
        assert abs(prob[r] - want[1]) <= 2.0 ** -23
    assert (ids[[0, 2, 3, 6, 7, 8, 9, 10, 11]] == -1).all() and ids[1] == 2999
    x2 = np.full((2, 70000), np.finfo(np.float32).min, np.float32)   # the same over several blocks
    x2[1, 69999] = 0.0
    check_draw(be, x2, k=35001, u=np.float32(0.9999))
    assert draw(be, x2, u=[0.5, 0.5], with_extras=False)[0].tolist()[1] == 69999


def test_sampling_the_largest_vocabulary(be):
    x = (np.random.default_rng(5).standard_normal((2, 360448)) * 2).astype(np.float32)
    check_draw(be, x, 0.9, [0, 300], [0.9, 0.8], 0.0, seed=6)
    with pytest.raises(BackendError):
        draw(be, np.zeros((1, 360449), np.float32), u=[0.5])


def test_sampling_does_not_depend_on_the_batch(be):
    """A row answers the same alone (more blocks to a row) and in a crowd."""
    x = np.random.default_rng(3).standard_normal((200, 40000)).astype(np.float32)
    u = np.random.default_rng(4).random(200).astype(np.float32)
    many = draw(be, x, 0.9, None, 0.95, None, u)
    for r in (0, 77, 199):
        one = draw(be, x[r:r + 1], 0.9, None, 0.95, None, u[r:r + 1])
        assert all(np.array_equal(a[r:r + 1], b) for a, b in zip(many, one))


# ------------------------------------------------------------------------------------------ caller-owned memory, graphs, a whole step

def test_imported_memory_and_stream_order(be):
    torch = pytest.importorskip("torch")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(64, 1 << 20, device="cuda")
        x = (big.sum(1, keepdim=True) * 0 + torch.randn(64, 5000, device="cuda")).contiguous()      # written late on another stream
        u = torch.rand(64, device="cuda")
        ids = torch.full((64,), -7, dtype=torch.int32, device="cuda")
    hx, hu, hids = be.import_tensor(x), be.import_tensor(u), be.import_tensor(ids)
    be.wait_stream(side.cuda_stream)
    sample_tokens(be, hx, SampleArgs(64, 5000), hu, hids)
    be.stream_wait(side.cuda_stream)
    with torch.cuda.stream(side):
        got = ids.clone()
    side.synchronize()
    xs, us = x.cpu().numpy(), u.cpu().numpy()
    assert got.cpu().tolist() == [sample_ref(xs[r], 1.0, 0, 1.0, 0.0, float(us[r]))[0] for r in range(64)]
    for h in (hx, hu, hids):
        h.release()
    assert float(x[0, 0]) == float(xs[0, 0])                          # the memory is still the tensor's
    with pytest.raises(BackendError):
        be.import_device(np.zeros(4).ctypes.data, 32)                 # host memory
    with pytest.raises(BackendError):
        be.import_device(0, 32)
    with pytest.raises(ValueError):
        be.import_tensor(torch.zeros(4, 6, device="cuda").t())
    empty = be.import_device(0, 0)
    assert empty.device_ptr == 0


class Step:
    """One serving step on the device: append with rotation, attention, a linear layer as the head, sampling."""

    def __init__(self, be, bt, vocab=512, n_pos=1024):
        rng = np.random.default_rng(20)
        self.be, self.bt, self.vocab = be, bt, vocab
        e = bt.heads * bt.dh
        self.qkv = rng.standard_normal((bt.rows, e + 2 * bt.kv_heads * bt.dh)).astype(np.float32)
        w = (rng.standard_normal((vocab, e)) * 0.3).astype(np.float32)
        self.wq, self.ws = O.quantize_i8_per_row(w)
        self.u = rng.random(bt.rows).astype(np.float32)
        self.cos, self.sin = P.rope_table(10000.0, bt.dh, n_pos)
        self.tables, self.starts, self.lens = index_buffers(be, bt)
        self.kp, self.vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
        self.d = {n: be.upload(getattr(self, n)) for n in ("qkv", "cos", "sin", "wq", "ws", "u")}
        self.q, self.o = be.alloc_zeroed((bt.rows, e)), be.alloc_zeroed((bt.rows, e))
        self.logits, self.ids = be.alloc_zeroed((bt.rows, vocab)), be.alloc_zeroed((bt.rows,), np.int32)
        self.scale = bt.dh ** -0.5
        self.aa = P.RopeAppendArgs(layout_of(bt), bt.batch, bt.rows, bt.heads, bt.kv_heads, bt.width, bt.dh, n_pos)
        self.ca = P.PagedChunkArgs(layout_of(bt), bt.batch, bt.rows, bt.rows, bt.width * bt.block, bt.heads, bt.kv_heads, bt.width, self.scale)
        self.sa = SampleArgs(bt.rows, vocab)
        self.wsp = be.alloc_zeroed((max(16, P.paged_chunk_workspace(be, self.ca)),), np.uint8)

    def run(self):
        d, be = self.d, self.be
        P.rope_paged_kv_append(be, d["qkv"], d["cos"], d["sin"], self.tables, self.starts, self.lens, self.kp, self.vp, self.aa, self.q)
        P.paged_chunk_attention(be, self.q, self.kp, self.vp, self.tables, self.starts, self.lens, self.ca, self.wsp, self.o)
        be.linear_forward_device_into(self.o, self.bt.rows, self.bt.heads * self.bt.dh, d["wq"], 0, d["ws"], 0, None, 0, self.vocab, 0, self.logits)
        sample_tokens(be, self.logits, self.sa, d["u"], self.ids)

    def check(self, qkv):
        """The operators in a row against the plain forms, each on the operands that the device handed to it."""
        bt = self.bt
        n = int(bt.q_starts[-1])
        (rq, rk, rv), (mq, _, _) = append_ref(bt, qkv, self.cos, self.sin, bt.dh, False)
        q = self.q.numpy()
        assert (np.abs(q[:n] - rq[:n]) <= mq[:n] * 2.0 ** -23).all()
        after = Batch(bt.new, bt.total, bt.heads, bt.kv_heads, bt.dh, bt.block, pad_rows=bt.rows - n)
        after.tables, after.k, after.v = bt.tables, down(self.kp, bt.k.shape, True), down(self.vp, bt.v.shape, True)
        assert np.abs(after.k - rk).max() < 0.05 and np.array_equal(after.v, bf16(rv).reshape(after.v.shape))
        ref, bound = attention_ref(after, q, self.scale)
        o = self.o.numpy()
        assert (np.abs(o[:n] - ref[:n]) <= bound[:n] + 2.0 ** -23 * np.abs(ref[:n])).all()
        logits, ids = self.logits.numpy(), self.ids.numpy()
        assert [int(i) for i in ids[:n]] == [sample_ref(logits[r], 1.0, 0, 1.0, 0.0, float(self.u[r]))[0] for r in range(n)]


def test_a_serving_step_of_the_operators_together(be):
    st = Step(be, Batch([7, 1, 33, 1], [7, 100, 64, 17], heads=8, kv_heads=2, dh=128, seed=21, pad_rows=2))
    st.run()
    st.check(st.qkv)


def test_a_captured_step_replays_with_other_inputs(be):
    torch = pytest.importorskip("torch")
    st = Step(be, Batch([7, 1, 33, 1], [7, 100, 64, 17], heads=8, kv_heads=2, dh=128, seed=22, pad_rows=6, spare_blocks=8))
    st.run()                                                          # modules, attributes and the linear layer's scratch
    be.synchronize_device()
    stream = torch.cuda.ExternalStream(be.stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        st.run()
    # another batch of the same capacity: other lengths, other chunks, one sequence less with rows
    bt = Batch([5, 0, 40, 2], [90, 3, 41, 112], heads=8, kv_heads=2, dh=128, seed=23, pad_rows=1)
    assert bt.rows == st.bt.rows and bt.blocks <= st.bt.blocks + 8
    big = st.bt
    bt.blocks, bt.width = big.blocks, big.width
    order = np.random.default_rng(1).permutation(big.blocks).astype(np.uint32)
    bt.tables = np.full((4, big.width), P.SENTINEL, np.uint32)
    at = 0
    for b, t in enumerate(bt.total):
        used = min(-(-t // 16), big.width)
        bt.tables[b, :used] = order[at:at + used]
        at += used
    assert at <= big.blocks
    bt.k, bt.v = big.k, big.v
    qkv = np.random.default_rng(24).standard_normal(st.qkv.shape).astype(np.float32)
    be.upload_into(bt.tables, st.tables)
    be.upload_into(bt.q_starts, st.starts)
    be.upload_into(bt.seq_lens, st.lens)
    be.upload_into(bt.pool_array(bt.k), st.kp)
    be.upload_into(bt.pool_array(bt.v), st.vp)
    be.upload_into(qkv, st.d["qkv"])
    be.synchronize_device()
    with torch.cuda.stream(stream):
        graph.replay()
    be.synchronize_device()
    st.bt = bt
    st.check(qkv)
    del graph


def make_small_decoder(be, batch):
    from fandhe_ai_b200.decoder import Decoder, DecoderConfig

    cfg = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, d_ff=512, vocab=512)
    dec = Decoder(be, DecoderConfig(**cfg, max_batch=batch, max_seq_len=32))
    dec.init_random(3, 0.05)
    return dec


def test_decoder_draws_on_the_device_and_feeds_what_it_drew(be):
    """Two decoders with the same weights: one draws on the device and feeds its ids without the host, the other gets the plain form's
    draws from its own logits as host ids.  They must stay together."""
    rng = np.random.default_rng(30)
    batch, steps = 3, 10
    a, b = make_small_decoder(be, batch), make_small_decoder(be, batch)
    try:
        for dec in (a, b):
            dec.begin(batch, [steps + 2] * batch)
        ids = np.array([3, 77, 400], np.int32)
        a.step(ids, want_next=False)
        b.step(ids)
        t, k, p, m = np.array([0.7, 1.5, 0.0]), np.array([0, 40, 0]), np.array([0.9, 1.0, 1.0]), 0.02
        for s in range(steps):
            u = rng.random(batch).astype(np.float32)
            logits = b.logits()
            assert np.array_equal(logits, a.logits())
            want = [sample_ref(logits[r], float(np.float32(t[r])), int(k[r]), float(np.float32(p[r])), float(np.float32(m)), float(u[r]))[0] for r in range(batch)]
            got = a.sample(u, t, k, p, m, want_ids=s % 2 == 0)
            if got is not None:
                assert got.tolist() == want
            a.step(None, want_next=False)
            b.step(np.array(want, np.int32))
        for bad in (dict(uniform=[0.1, 1.0, 0.2]), dict(uniform=0.1, temperature=-1.0), dict(uniform=0.1, top_p=np.nan)):
            with pytest.raises(BackendError):
                a.sample(**bad)
    finally:
        a.close()
        b.close()


def test_decoder_sample_needs_a_step(be):
    dec = make_small_decoder(be, 2)
    try:
        dec.begin(2, [4, 4])
        with pytest.raises(BackendError):
            dec.sample(0.5)
    finally:
        dec.close()


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_long_chunks_among_single_tokens(be, dh, io_bf16):
    """Chunks, single tokens and sequences without new ones in one batch: items of every kind in one launch."""
    check_attention(be, Batch([1, 200, 1, 0, 3, 1, 1, 1, 2, 1], [40, 330, 600, 5, 3, 1, 129, 300, 2, 17], heads=8, kv_heads=2, dh=dh, seed=17, pad_rows=2), io_bf16)
    # and with the keys of a row shared out
    check_attention(be, Batch([1, 40, 1, 1, 1, 1], [3000, 2100, 60, 900, 1, 5000], heads=4, kv_heads=1, dh=dh, seed=18), io_bf16)
    check_attention(be, Batch([1] * 20 + [90], [33] * 20 + [90], heads=4, kv_heads=4, dh=dh, seed=19), io_bf16)
