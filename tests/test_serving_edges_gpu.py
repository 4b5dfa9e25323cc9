"""Serving operators of a ragged batch on the GPU at their edges: batches of short items, unusual values, other threads and streams."""
import numpy as np
import pytest

from fandhe_ai_b200 import BF16, F32, Backend, BackendError
from fandhe_ai_b200 import paged_kv as P

from fandhe_ai_b200.decoder import SampleArgs, sample_tokens

from serving_ref import Batch, attention_ref, bf16, sample_ref
from test_serving_gpu import check_attention, check_draw, down, draw, layout_of, make_small_decoder, run_attention, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_many_items_of_one_tile(be, dh, io_bf16):
    """Sequences of one key tile, hundreds of items to a block's turn: one of the two slots has nothing to multiply in any of them."""
    check_attention(be, Batch([1] * 700, [1 + 13 * i % 128 for i in range(700)], heads=4, kv_heads=2, dh=dh, seed=31), io_bf16)
    new = [11 + 7 * i % 20 for i in range(200)]
    check_attention(be, Batch(new, [n + 5 * i % 97 for i, n in enumerate(new)], heads=4, kv_heads=4, dh=dh, seed=32), io_bf16)
    # one tile and several tiles in turn, more rows than the variant for few rows takes
    new = [12, 60, 12, 33] * 30
    check_attention(be, Batch(new, [n + [0, 200, 90, 600][i % 4] for i, n in enumerate(new)], heads=2, kv_heads=1, dh=dh, seed=33), io_bf16)


# ------------------------------------------------------------------------------------------ device arrays that make no sense

def reported(be):
    with pytest.raises(BackendError) as e:
        be.synchronize_device()
    return e.value.message


BAD_STARTS = [
    dict(starts=[0, 100, 2, 3], lens=[100, 60, 40], rows=110, dh=64),        # the second sequence ends before it starts
    dict(starts=[0, 100, 2, 3], lens=[100, 60, 40], rows=110, dh=80),
    dict(starts=[0, 3, 1, 2], lens=[4000, 4000, 4000], rows=6, dh=128),      # the same with the keys of a row shared out and joined
    dict(starts=[0, 3, 1, 2], lens=[4000, 4000, 4000], rows=6, dh=40),
    dict(starts=[0, 4, 9], lens=[40, 40], rows=8, dh=64),                    # ends behind the last row
    dict(starts=[0, 4, 9], lens=[40, 40], rows=8, dh=80),
    dict(starts=[0, 4, 4, 8], lens=[40, 70, 40], rows=8, dh=64, max_len=64),  # too long, and without a new token
    dict(starts=[0, 4, 4, 8], lens=[40, 70, 40], rows=8, dh=80, max_len=64),
]


@pytest.mark.parametrize("case", BAD_STARTS)
def test_starts_that_make_no_sense_are_reported(case):
    be = Backend(0)
    try:
        starts, lens, rows, dh = case["starts"], case["lens"], case["rows"], case["dh"]
        bt = Batch([1] * len(lens), lens, heads=4, kv_heads=2, dh=dh, seed=40)
        q = be.upload(np.random.default_rng(1).standard_normal((rows, 4 * dh)).astype(np.float32))
        tables, st, sl = be.upload(bt.tables), be.upload(np.array(starts, np.uint32)), be.upload(bt.seq_lens)
        kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
        layout = P.PagedKvLayout(bt.blocks, bt.block, 2 * dh, BF16)
        most = case.get("max_len", max(lens))
        args = P.PagedChunkArgs(layout, len(lens), rows, min(100, most), most, 4, 2, bt.width, 0.1)
        need = P.paged_chunk_workspace(be, args)
        ws = be.upload(np.zeros(max(16, need), np.uint8))
        out = be.upload(np.full((rows, 4 * dh), 7.0, np.float32))
        P.paged_chunk_attention(be, q, kp, vp, tables, st, sl, args, ws, out)
        assert "0x205" in reported(be)
    finally:
        be.close()
    be = Backend(0)
    try:
        qkv = be.upload(np.random.default_rng(2).standard_normal((rows, 8 * dh)).astype(np.float32))
        tables, st, sl = be.upload(bt.tables), be.upload(np.array(starts, np.uint32)), be.upload(bt.seq_lens)
        kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
        cos, sin = (be.upload(x) for x in P.rope_table(10000.0, dh, max(lens) + 1))
        width = case["max_len"] // bt.block if "max_len" in case else bt.width
        t2 = be.upload(np.ascontiguousarray(bt.tables[:, :width]))
        args = P.RopeAppendArgs(layout, len(lens), rows, 4, 2, width, dh, max(lens) + 1)
        P.rope_paged_kv_append(be, qkv, cos, sin, t2, st, sl, kp, vp, args, be.upload(np.zeros((rows, 4 * dh), np.float32)))
        assert "0x205" in reported(be)
    finally:
        be.close()


@pytest.mark.parametrize("dh", [64, 80, 128])
def test_starts_that_make_no_sense_leave_the_rest_alone(dh):
    """Memory of torch, which can be read after the error: rows of no sequence, guard rows and the workspace's guard keep what they held."""
    torch = pytest.importorskip("torch")
    be = Backend(0)
    try:
        lens, rows = [4000, 4000, 4000], 6
        bt = Batch([1] * 3, lens, heads=4, kv_heads=2, dh=dh, seed=41)
        layout = P.PagedKvLayout(bt.blocks, bt.block, 2 * dh, BF16)
        args = P.PagedChunkArgs(layout, 3, rows, 100, 4000, 4, 2, bt.width, 0.1)
        need = P.paged_chunk_workspace(be, args)
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        out = torch.full((rows + 8, 4 * dh), 7.0, device="cuda")
        torch.cuda.synchronize()
        up = lambda x: be.upload(np.ascontiguousarray(x))
        P.paged_chunk_attention(be, up(bt.q[:1].repeat(rows, 0)), up(bt.pool_array(bt.k)), up(bt.pool_array(bt.v)), up(bt.tables),
                                up(np.array([0, 3, 1, 2], np.uint32)), up(bt.seq_lens), args, be.import_tensor(ws), be.import_tensor(out))
        assert "0x205" in reported(be)
        assert bool((out[3:] == 7.0).all()) and bool((ws[need:] == 0x5A).all())
    finally:
        be.close()


# ------------------------------------------------------------------------------------------ streams

def test_stream_order_both_ways_again_and_again(be):
    """Two streams of another library in turn, each ordered against the context's: every call sees the values that its own stream wrote
    last, although all calls share the context's event."""
    torch = pytest.importorskip("torch")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    x, ids, u = [torch.zeros(4, 5000, device="cuda") for _ in streams], [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in streams], torch.zeros(4, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    hx, hid, hu = [be.import_tensor(t) for t in x], [be.import_tensor(t) for t in ids], be.import_tensor(u)
    got = []
    for i in range(40):
        j = i % 2
        with torch.cuda.stream(streams[j]):
            if i % 8 == j:
                _ = big @ big
            x[j].fill_(-1.0)
            x[j][:, 37 * i + j] = 5.0
            be.wait_stream(streams[j].cuda_stream)
            sample_tokens(be, hx[j], SampleArgs(4, 5000), hu, hid[j], top_k=None, temperature=hu)       # temperature 0: the maximum
            be.stream_wait(streams[j].cuda_stream)
            got.append(ids[j].clone())
            x[j].zero_()
    torch.cuda.synchronize()
    assert [g.tolist() for g in got] == [[37 * i + i % 2] * 4 for i in range(40)]


def test_stream_order_inside_a_captured_graph(be):
    """A stream of another library is captured; the context joins the capture for one call and hands over again."""
    torch = pytest.importorskip("torch")
    x, ids, u = torch.zeros(4, 5000, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    at = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    hx, hid, hu = be.import_tensor(x), be.import_tensor(ids), be.import_tensor(u)
    side = torch.cuda.Stream()

    def step():
        x.fill_(-1.0)
        x.scatter_(1, at, 5.0)
        be.wait_stream(torch.cuda.current_stream().cuda_stream)
        sample_tokens(be, hx, SampleArgs(4, 5000), hu, hid, temperature=hu)
        be.stream_wait(torch.cuda.current_stream().cuda_stream)
        return ids * 2

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        twice = step()
    for i in (3, 4999, 0, 77):
        at.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert twice.tolist() == [2 * i] * 4
    be.wait_stream(side.cuda_stream)             # and outside a capture again
    sample_tokens(be, hx, SampleArgs(4, 5000), hu, hid, temperature=hu)
    assert hid.numpy().tolist() == [77] * 4
    del graph
def measured_cases():
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("measured_cases", Path(__file__).resolve().parents[1] / "perf" / "operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_measured_calls_are_ordered_with_the_callers_stream(be):
    """perf/operators.py hands out tensors of torch: its calls wait for what the current stream has still to write, and work that
    the caller puts behind them sees finished results - without a wait of the host in between."""
    torch = pytest.importorskip("torch")
    m = measured_cases()
    m.own = True
    case = dict(op="attention", dtype="bf16", seqs=2, chunked=2, chunk_lo=900, chunk_hi=1000, step=1, prefix_lo=0, prefix_hi=0, lens=1,
                heads=8, kv_heads=8, head_dim=128, block=16)
    st = m.prepare(case, 5)
    torch.cuda.synchronize()
    want = m.run(st)["out"].clone()
    torch.cuda.synchronize()
    big, q = torch.randn(8192, 8192, device="cuda"), st["q"].clone()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        st["q"].zero_()
        st["out"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(4):
                big = big @ big * 1e-4                       # some milliseconds before the queries are there
            st["q"].copy_(q)
            got = m.run(st)["out"].clone()
            st["q"].zero_()                                  # and gone again as soon as the call's place in the stream is past
        stream.synchronize()
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------ sampling

@pytest.mark.parametrize("min_p", [1e-3, 1e-6, 1e-10, 1e-14, 1e-18, 1e-30])
@pytest.mark.parametrize("vocab", [50, 5000, 128256])
def test_sampling_min_p_is_compared_with_the_weight_itself(be, vocab, min_p):
    """Tokens one step of f32 apart around the border, far below the resolution of the sums."""
    m = np.float32(min_p)
    rows = 3
    x = np.full((rows, vocab), -np.inf, np.float32)
    border = np.float32(np.log(float(m)))
    near = [border]
    for _ in range(4):
        near = [np.nextafter(near[0], np.float32(-np.inf)), *near, np.nextafter(near[-1], np.float32(0))]
    at = np.random.default_rng(vocab).permutation(vocab)[:len(near) + 2]
    for r in range(rows):
        x[r, at[:-2]] = near
        x[r, at[-2]] = 0.0
        x[r, at[-1]] = border * 2                                   # far below the border
    # f64 exponentials differ by 2^-50; a step of f32 at the border is at least 2^-23 of the logit, and the weight moves as much
    assert np.abs(np.exp(np.float64(near)) / float(m) - 1).min() > 1e-9
    want = sample_ref(x[0], 1.0, 0, 1.0, float(m), 0.0)
    for kw in (dict(), dict(k=vocab), dict(k=len(at) + 1)):
        ids, prob, kept = draw(be, x, m=m, u=[0.0, 0.3, 0.9999999], **kw)
        assert kept.tolist() == [want[2]] * 3 and want[2] not in (1, len(at))
        assert ids[0] == want[0] and ids[1:].tolist() == [sample_ref(x[0], 1.0, 0, 1.0, float(m), u)[0] for u in (float(np.float32(0.3)), float(np.float32(0.9999999)))]


@pytest.mark.parametrize("vocab,as_bf16", [(32767, True), (32768, True), (65536, True), (131072, True), (262144, True), (262144, False)])
def test_sampling_vocabularies_that_are_powers_of_two(be, vocab, as_bf16):
    """The longest runs of logits a thread has to go through, 65 of them, and the borders of the survivors among them."""
    rng = np.random.default_rng(vocab)
    rows = 6
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    x[0, [0, 63, 64, 65, vocab // 2, vocab - 1]] = 12.0               # first, last and the borders of a run
    x[1, 64::65] += 4.0                                               # the last element of every run
    x[2] = -np.inf
    x[2, vocab - 70:] = np.linspace(-3, 3, 70)
    check_draw(be, x, [1.0, 0.8, 1.0, 0.7, 1.0, 1.1], [0, 200, 0, 50, 1000, 0], [0.9, 0.95, 0.9, 1.0, 0.7, 0.99],
               [0.0, 0.0, 0.05, 0.0, 0.02, 0.01], seed=vocab + 3, as_bf16=as_bf16)


def test_threads_that_use_kernels_for_the_first_time_at_once():
    """Contexts of their own, vocabularies in a different order each: a smaller one must not take the shared memory of a larger one
    away.  In a process of its own, whose kernels nobody has used yet."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys, threading
import numpy as np
from fandhe_ai_b200 import Backend
from fandhe_ai_b200.decoder import SampleArgs, sample_tokens
sizes = [360448, 20, 128256, 300000, 4097, 50000, 200000, 1000]
start, failed = threading.Barrier(4), []
def work(k):
    be = Backend(0)
    bufs = [(be.upload(np.eye(1, v, v // 2, dtype=np.float32) * 50), v) for v in sizes[2 * k:] + sizes[:2 * k]]
    u, ids = be.upload(np.zeros(1, np.float32)), be.alloc_zeroed((1,), np.int32)
    be.synchronize_device()
    start.wait()
    try:
        for _ in range(30):
            for x, v in bufs:
                sample_tokens(be, x, SampleArgs(1, v), u, ids)
        for x, v in bufs:
            sample_tokens(be, x, SampleArgs(1, v), u, ids, temperature=u)
            assert ids.numpy()[0] == v // 2
    except Exception as e:
        failed.append((k, v, e))
    be.close()
threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
[t.start() for t in threads]; [t.join() for t in threads]
assert not failed, failed
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------ infinities and NaN that a token sees

# the forms of the attention: few rows, at most 32 rows, 128 rows, 256 rows, keys shared out and joined, the general kernel
FORMS = [
    dict(new=[1, 2], total=[300, 140]),
    dict(new=[1, 1], total=[300, 40], dh=64),
    dict(new=[8], total=[300]),
    dict(new=[16], total=[300], dh=64, heads=4, kv_heads=2),
    dict(new=[32], total=[500]),
    dict(new=[60], total=[400], dh=64),
    dict(new=[80, 70], total=[500, 310], heads=8, kv_heads=2),
    dict(new=[3], total=[6000], heads=4, kv_heads=1),
    dict(new=[40], total=[4000], heads=4, kv_heads=1),
    dict(new=[90], total=[3000], heads=8, kv_heads=2, dh=64),
    dict(new=[5, 1], total=[200, 3], dh=80),
    dict(new=[5, 1], total=[200, 3], pool_bf16=False),
]


def check_non_finite(be, bt, io_bf16, scale, places):
    """`places`: (key, element, value) of KV head 0 of sequence 0.  Where one token sees them, the element is their sum; the others do
    not notice."""
    blk, off = bt.places(0)
    clean = bt.v.copy()
    for key, e, value in places:
        bt.v[blk[key], off[key], e] = value
    q = bf16(bt.q) if io_bf16 else bt.q
    got = run_attention(be, bt, q, io_bf16, scale)
    bt.v, dirty = clean, bt.v
    ref, bound = attention_ref(bt, q, scale, split_terms=not io_bf16)
    g, first = bt.heads // bt.kv_heads, bt.total[0] - bt.new[0]
    step = 2.0 ** -8 if io_bf16 else 2.0 ** -24
    want = ref.copy()
    for i in range(bt.new[0]):
        for key, e, value in places:
            if key <= first + i:
                for h in range(g):
                    at = h * bt.dh + e
                    with np.errstate(invalid="ignore"):      # inf - inf
                        want[i, at] = value + (want[i, at] if not np.isfinite(want[i, at]) else 0.0)
    touched = ~np.isfinite(want)
    assert touched.any() and (np.abs(got - ref) <= bound + step * 1.001 * (np.abs(ref) + bound))[~touched].all()
    assert np.array_equal(got[touched], want[touched].astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", FORMS)
def test_attention_infinities_that_every_token_sees(be, case, io_bf16):
    inf, dh = np.inf, case.get("dh", 128)
    for key in (0, 2, 37, 130, 200):
        if key < case["total"][0] - case["new"][0]:
            check_non_finite(be, Batch(seed=50, **case), io_bf16, dh ** -0.5, [(key, 3, inf), (key, 40, -inf), (key, 41, np.nan), (0, dh - 1, inf)])
    key = min(150, case["total"][0] - case["new"][0] - 1)
    check_non_finite(be, Batch(seed=51, **case), io_bf16, dh ** -0.5, [(0, 7, inf), (key, 7, inf), (1, 8, inf), (key, 8, -inf)])
    # weights that vanish next to the largest, and a key that a later maximum scales down
    check_non_finite(be, Batch(seed=52, q_scale=30.0, **case), io_bf16, dh ** -0.5, [(0, 7, inf), (key, 9, -inf), (key // 2, 10, inf)])


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", FORMS)
def test_attention_nan_of_a_key_reaches_every_token_that_sees_it(be, case, io_bf16):
    for key in (0, case["total"][0] - 1):
        bt = Batch(seed=53, **case)
        blk, off = bt.places(0)
        bt.k[blk[key], off[key], 5] = np.nan
        got = run_attention(be, bt, bf16(bt.q) if io_bf16 else bt.q, io_bf16, 0.1)
        first, g = bt.total[0] - bt.new[0], bt.heads // bt.kv_heads
        sees = np.zeros(got.shape, bool)
        sees[max(0, key - first):bt.new[0], :g * bt.dh] = True
        assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", FORMS)
def test_attention_infinities_of_a_key(be, case, io_bf16):
    """A score of -inf has no weight; one of +inf leaves no number (inf - inf)."""
    for key, value, scale in ((0, np.inf, 0.1), (2, -np.inf, 0.1), (min(150, case["total"][0] - case["new"][0] - 1), np.inf, -0.1)):
        bt = Batch(seed=54, **case)
        blk, off = bt.places(0)
        q = bf16(bt.q) if io_bf16 else bt.q
        n, t, dh, g = bt.new[0], bt.total[0], bt.dh, bt.heads // bt.kv_heads
        ref, bound = attention_ref(bt, q, scale, split_terms=not io_bf16)
        ks = bt.k[blk, off].astype(np.float64).reshape(t, bt.kv_heads, dh)[:, 0]
        vs = bt.v[blk, off].astype(np.float64).reshape(t, bt.kv_heads, dh)[:, 0]
        bt.k[blk[key], off[key], 6] = value
        got = run_attention(be, bt, q, io_bf16, scale)
        step = 2.0 ** -8 if io_bf16 else 2.0 ** -24
        numbers = 0
        for i in range(n):
            keep = np.array([j for j in range(t - n + i + 1) if j != key])
            for h in range(g):
                sl = slice(h * dh, (h + 1) * dh)
                if q[i, h * dh + 6] * value * scale > 0:
                    assert np.isnan(got[i, sl]).all()
                    continue
                s = ks[keep] @ q[i, sl].astype(np.float64) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                ds = (dh + 8) * 2.0 ** -23 * abs(scale) * (np.abs(ks[keep]) @ np.abs(q[i, sl].astype(np.float64))).max()
                rel = np.expm1(2 * ds + 2.0 ** -21) + (2.0 ** -8 if io_bf16 else 2.0 ** -16) + 2 * len(keep) * 2.0 ** -23
                lim = 2 * rel * (p @ np.abs(vs[keep]))
                want = p @ vs[keep]
                assert (np.abs(got[i, sl] - want) <= lim + step * 1.001 * (np.abs(want) + lim)).all()
                numbers += 1
        rest = np.ones(got.shape, bool)
        rest[:n, :g * dh] = False
        assert (np.abs(got - ref) <= bound + step * 1.001 * (np.abs(ref) + bound))[rest].all()
        assert numbers > 0 or n * g < 4


# ------------------------------------------------------------------------------------------ the decoder's own draw

def step_rows(dec, ids, active):
    a, nxt = np.array(active, np.uint8), np.empty(len(active), np.int32)
    c = np.ascontiguousarray(ids, np.int32) if ids is not None else None
    P.check(P.lib().b200_decoder_step_rows(dec._h, c.ctypes.data if c is not None else None, a.ctypes.data, nxt.ctypes.data))
    return nxt


def test_decoder_draws_for_the_rows_that_took_part(be):
    """A row that sat the step out needs no valid parameters and keeps its id; the others draw as ever."""
    dec = make_small_decoder(be, 3)
    try:
        dec.begin(3, [12] * 3)
        dec.step(np.array([3, 77, 400], np.int32))
        nan = float("nan")
        for active, uniform, temperature, top_p in (([1, 0, 1], [0.3, nan, 0.7], [1.0, -1.0, 1.3], [0.9, nan, 1.0]),
                                                    ([0, 1, 0], [2.0, 0.9, -1.0], [nan, 0.8, nan], [nan, 0.5, nan])):
            left = step_rows(dec, [5, 6, 7], active)
            logits = dec.logits()
            got = dec.sample(uniform, temperature, top_p=top_p)
            for r in range(3):
                want = left[r]
                if active[r]:
                    want = sample_ref(logits[r], float(np.float32(temperature[r])), 0, float(np.float32(top_p[r])), 0.0, float(np.float32(uniform[r])))[0]
                assert got[r] == want
        with pytest.raises(BackendError, match="row 1: uniform"):
            dec.sample([0.1, nan, 0.1])                       # the row that takes part
        step_rows(dec, None, [1, 1, 1])
        with pytest.raises(BackendError):
            dec.sample([0.1, 0.1, nan])
        assert (dec.sample([0.1, 0.1, 0.1]) >= 0).all()
    finally:
        dec.close()


# ------------------------------------------------------------------------------------------ arguments

@pytest.mark.parametrize("adjacent", [False, True])
def test_append_without_rotation_takes_no_tables(be, adjacent):
    bt = Batch([3, 2], [20, 2], heads=4, kv_heads=1, dh=64, seed=5)
    qkv = np.random.default_rng(6).standard_normal((5, 6 * 64)).astype(np.float32)
    tables, st, sl = be.upload(bt.tables), be.upload(bt.q_starts), be.upload(bt.seq_lens)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    layout = P.PagedKvLayout(bt.blocks, bt.block, 64, BF16)
    for rotary, n_pos in ((0, 0), (0, 77)):
        q = be.alloc_zeroed((5, 256))
        P.rope_paged_kv_append(be, be.upload(qkv), None, None, tables, st, sl, kp, vp, P.RopeAppendArgs(layout, 2, 5, 4, 1, bt.width, rotary, n_pos, adjacent), q)
        assert np.array_equal(q.numpy(), qkv[:, :256])
    with pytest.raises(BackendError) as e:
        P.rope_paged_kv_append(be, be.upload(qkv), None, None, tables, st, sl, kp, vp, P.RopeAppendArgs(layout, 2, 5, 4, 1, bt.width, 64, 32, adjacent), q)
    assert e.value.kind == "InvalidArgument"


def test_overlapping_memory_is_refused(be):
    bt = Batch([4, 4], [100, 60], heads=4, kv_heads=2, seed=16)
    tables, st, sl = be.upload(bt.tables), be.upload(bt.q_starts), be.upload(bt.seq_lens)
    kp, vp = be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v))
    layout = P.PagedKvLayout(bt.blocks, bt.block, 256, BF16)
    args = P.PagedChunkArgs(layout, 2, 8, 4, 100, 4, 2, bt.width, 0.1)
    need = P.paged_chunk_workspace(be, args)
    big = be.alloc_zeroed((1 << 20,))
    row = 512 * 4

    def refused(call, *a, **kw):
        with pytest.raises(BackendError) as e:
            call(be, *a, **kw)
        assert e.value.kind == "InvalidArgument" and "overlap" in e.value.message

    ws, q, out = be.alloc_zeroed((max(16, need),), np.uint8), be.alloc_zeroed((8, 512)), be.alloc_zeroed((8, 512))
    refused(P.paged_chunk_attention, big, kp, vp, tables, st, sl, args, ws, big, q_off=0, out_off=row)
    wide = P.PagedChunkArgs(layout, 2, 8, 4, 100, 4, 2, bt.width, 0.1, q_stride=516)
    refused(P.paged_chunk_attention, big, kp, vp, tables, st, sl, wide, ws, big)                # the same start, rows apart
    refused(P.paged_chunk_attention, q, kp, big, tables, st, sl, args, ws, big, out_off=0)
    if need:
        refused(P.paged_chunk_attention, big, kp, vp, tables, st, sl, args, big, out)
        refused(P.paged_chunk_attention, q, kp, vp, tables, st, sl, args, big, big, out_off=16)
    cos, sin = (be.upload(x) for x in P.rope_table(1e4, 128, 200))
    ra = P.RopeAppendArgs(layout, 2, 8, 4, 2, bt.width, 128, 200)
    refused(P.rope_paged_kv_append, big, cos, sin, tables, st, sl, kp, vp, ra, big, q_out_off=7 * 1024 * 4)
    refused(P.rope_paged_kv_append, big, cos, sin, tables, st, sl, big, vp, ra, q)
    refused(P.rope_paged_kv_append, be.alloc_zeroed((8, 1024)), cos, sin, tables, st, sl, kp, kp, ra, q)
    refused(P.rope_paged_kv_append, be.alloc_zeroed((8, 1024)), cos, sin, tables, st, sl, kp, big, ra, big)
    assert not be.poisoned


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", FORMS)
def test_attention_in_place(be, case, io_bf16):
    bt = Batch(seed=60, pad_rows=2, **case)
    q = bf16(bt.q) if io_bf16 else bt.q
    want = run_attention(be, bt, q, io_bf16, 0.1)
    both = up(be, q, io_bf16)
    args = P.PagedChunkArgs(layout_of(bt), bt.batch, bt.rows, max(bt.new), max(bt.total), bt.heads, bt.kv_heads, bt.width, 0.1, BF16 if io_bf16 else F32)
    ws = be.alloc_zeroed((max(16, P.paged_chunk_workspace(be, args)),), np.uint8)
    tables, st, sl = be.upload(bt.tables), be.upload(bt.q_starts), be.upload(bt.seq_lens)
    P.paged_chunk_attention(be, both, be.upload(bt.pool_array(bt.k)), be.upload(bt.pool_array(bt.v)), tables, st, sl, args, ws, both)
    got, n = down(both, q.shape, io_bf16), bt.rows - 2
    assert np.array_equal(got[:n], want[:n]) and np.array_equal(got[n:], q[n:])


# ------------------------------------------------------------------------------------------ what only a small part of a number carries

# few rows, at most 32 rows (the three terms share the accumulator rows), more rows, keys shared out; heads of 64 and 128
TERMS = [dict(tokens=t, dh=dh, kv_heads=kv, group=g, total=n) for dh in (64, 128)
         for t, kv, g, n in ((2, 2, 4, 300), (1, 1, 8, 3000), (7, 2, 4, 300), (30, 2, 1, 290), (33, 2, 4, 400), (100, 1, 1, 300), (25, 2, 4, 2500))]


def weighted_pairs(case, x, at):
    """Sequences in which the keys at[b] (score 0, V 0) and at[b] + 1 (score -x[b], V 1) are the only ones with a weight."""
    n = len(x)
    bt = Batch([case["tokens"]] * n, [case["total"]] * n, heads=case["kv_heads"] * case["group"], kv_heads=case["kv_heads"], dh=case["dh"], seed=70)
    bt.k[:], bt.v[:], bt.q[:] = 0.0, 0.0, 0.0
    bt.q[:, ::bt.dh] = 1.0
    bt.k[..., ::bt.dh] = -1.0e4
    for b in range(n):
        blk, off = bt.places(b)
        bt.k[blk[at[b]], off[at[b]]] = 0.0
        bt.k[blk[at[b] + 1], off[at[b] + 1], ::bt.dh] = -x[b]
        bt.v[blk[at[b] + 1], off[at[b] + 1]] = 1.0
    return bt


@pytest.mark.parametrize("case", TERMS)
def test_attention_f32_weights_keep_all_their_bits(be, case):
    """out = w / (1 + w), w = e^-x: a weight cut to 16 bits is off by up to 2^-15 of it, which the bound does not allow.

    The bound, relative to out.  The argument of the exponential: c and its product round (2 2^-24 of |x| log2 e), times ln 2, twice where a
    partial maximum is scaled down: |x| 2^-22; the exponentials 2^-22 each, two: 2^-21; doubled, since out has w above and below.
    Then the sum, its reciprocal and the product (3 2^-24), and the accumulator, cut at each of its three terms (3 2^-23)."""
    first = case["total"] - case["tokens"]
    at = [p for p in (0, 3, 38, 62, 70, 94, 100, 126, 130, 165, 200, 228, 260) if p + 1 < first]
    rng = np.random.default_rng(71)
    x = bf16(rng.uniform(0.1, 3.5, 4 * len(at)).astype(np.float32))
    bt = weighted_pairs(case, x, at * 4)
    got = run_attention(be, bt, bt.q, False, 1.0)
    w = np.exp(-x.astype(np.float64))
    want = np.repeat(w / (1 + w), case["tokens"])[:, None]
    lim = want * (2 * (np.repeat(x, case["tokens"])[:, None] * 2.0 ** -22 + 2.0 ** -21) + 3 * 2.0 ** -24 + 3 * 2.0 ** -23)
    err = np.abs(got - want)
    # the test itself: weights without their third term would not pass
    w16 = (w.astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32).astype(np.float64)
    rest = (w.astype(np.float32) - w16).astype(np.float32)
    cut = w16 + (rest.view(np.uint32) & 0xFFFF0000).view(np.float32)
    assert (np.abs(cut / (1 + w) - w / (1 + w)) > 2 * lim[::case["tokens"], 0]).any()
    assert (err <= lim).all(), f"off by {(err / want).max():.3g}, allowed {(lim / want)[np.unravel_index(np.argmax(err / want), err.shape)[0], 0]:.3g}"


@pytest.mark.parametrize("case", TERMS)
def test_attention_f32_queries_keep_all_their_bits(be, case):
    """A score of 128 2^12 (q0 - q1) = +-1.5 that stands in the last bits of q0 alone: q0 = 1 + 2^-10 + d, q1 = 1 + 2^-10, d = +-0.75 2^-18.

    The products cancel at 2^12 in an accumulator that keeps 2^-23 of its largest addend; two cuts (the first element's product and
    the second's) are 2 2^-11, times the scale 0.125 in the score, e^0.125 - 1 in a weight, above and below: 0.29 of out.
    Without the third term the score is 0 and out is off by 1 - e^-1.5 = 0.78 of it, or e^1.5 - 1."""
    n = 3
    bt = Batch([case["tokens"]] * n, [case["total"]] * n, heads=case["kv_heads"] * case["group"], kv_heads=case["kv_heads"], dh=case["dh"], seed=72)
    bt.k[:], bt.v[:], bt.q[:] = 0.0, 0.0, 0.0
    d = np.where(np.arange(bt.rows) % 2 == 0, 1.0, -1.0) * 0.75 * 2.0 ** -18
    bt.q[:, 0::bt.dh] = (1 + 2.0 ** -10 + d)[:, None]
    bt.q[:, 1::bt.dh] = 1 + 2.0 ** -10
    for b, at in enumerate((0, 60, case["total"] - case["tokens"] - 1)):
        blk, off = bt.places(b)
        bt.k[blk[at], off[at], 0::bt.dh], bt.k[blk[at], off[at], 1::bt.dh] = 2.0 ** 12, -2.0 ** 12
        bt.v[blk[at], off[at]] = 1.0
    got = run_attention(be, bt, bt.q, False, 128.0)
    for row in range(bt.rows):
        see = case["total"] - case["tokens"] + 1 + row % case["tokens"]
        e = np.exp(128.0 * 2.0 ** 12 * d[row])
        want = e / (e + see - 1)
        assert (np.abs(got[row] - want) <= 0.29 * want).all()


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("case", FORMS)
def test_attention_a_token_sees_itself_and_not_the_next(be, case, io_bf16):
    """The values of the new tokens grow by half from one to the next, so that a row's own key is a third of what it sums up: one key
    too few or too many does not fit the bound of any form."""
    bt = Batch(seed=73, **case)
    for b in range(bt.batch):
        blk, off = bt.places(b)
        for i in range(bt.new[b]):
            at = bt.total[b] - bt.new[b] + i
            bt.v[blk[at], off[at]] = bf16(np.float32(300.0 * 1.5 ** i) * np.where(np.arange(bt.kv_heads * bt.dh) % 3 == 0, -1, 1).astype(np.float32))
    check_attention(be, bt, io_bf16, scale=0.02)
    # the test itself: the same rows with one key less are outside the bound
    q = bf16(bt.q) if io_bf16 else bt.q
    ref, bound = attention_ref(bt, q, 0.02, split_terms=not io_bf16)
    blk, off = bt.places(0)
    at = bt.total[0] - bt.new[0]
    bt.v[blk[at], off[at]] = 0.0
    less, _ = attention_ref(bt, q, 0.02, split_terms=not io_bf16)
    assert (np.abs(less[0] - ref[0]) > 2 * bound[0] + 2.0 ** -7 * np.abs(ref[0])).all()


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("seqs,chunk,cached", [(2, 512, 600), (2, 512, 8000), (4, 300, 4000), (48, 1, 16000)])
def test_attention_f32_error_does_not_grow_with_the_cache(dh, seqs, chunk, cached):
    """The tensor cores cut a sum at each addition: by half a last place on average, 2^-24 of it at most, always towards zero, so the
    parts add up.  An accumulator takes at most 48 additions before f32 additions go on with it, and a score 24 of its own size
    (rms 1.5, which moves the weights as much): (48 + 1.5 24) 2^-24 of the result.  Half that many again for all that rounds."""
    m = measured_cases()
    m.own = True
    case = dict(op="attention", dtype="f32", seqs=seqs, chunked=seqs, chunk_lo=chunk, chunk_hi=chunk, step=1, prefix_lo=cached, prefix_hi=cached,
                lens=2, heads=32, kv_heads=8, head_dim=dh, block=16)
    out, want = m.run(m.prepare(case, 3))["out"].double(), m.exact(case, 3)["out"]
    assert float((out - want).norm() / want.norm()) <= 1.5 * (48 + 1.5 * 24) * 2.0 ** -24


# ------------------------------------------------------------------------------------------ large and crowded

@pytest.mark.parametrize("dh,kv_heads,pool_bf16", [(128, 8, True), (64, 16, True), (80, 8, True), (128, 4, False)])
def test_pools_whose_offsets_pass_32_bits(be, dh, kv_heads, pool_bf16):
    """The same batch in the first blocks of a pool and in its last ones, more than 2^31 elements further on."""
    torch = pytest.importorskip("torch")
    block, ekv = 16, dh * kv_heads
    blocks = (1 << 31) // (block * ekv) + 200
    dtype = torch.bfloat16 if pool_bf16 else torch.float32
    bt = Batch([70, 1, 9], [500, 333, 9], heads=kv_heads * 2, kv_heads=kv_heads, dh=dh, pool_bf16=pool_bf16, seed=80)
    kp, vp = (torch.empty(blocks, block, ekv, dtype=dtype, device="cuda") for _ in range(2))
    assert kp.numel() > 1 << 31
    qkv = torch.randn(bt.rows, (bt.heads + 2 * kv_heads) * dh, device="cuda")
    cos, sin = (torch.from_numpy(x).cuda() for x in P.rope_table(1e4, dh, 600))
    layout = P.PagedKvLayout(blocks, block, ekv, BF16 if pool_bf16 else F32)
    aa = P.RopeAppendArgs(layout, bt.batch, bt.rows, bt.heads, kv_heads, bt.width, dh, 600)
    ca = P.PagedChunkArgs(layout, bt.batch, bt.rows, max(bt.new), max(bt.total), bt.heads, kv_heads, bt.width, 0.1)
    ws = torch.zeros(max(16, P.paged_chunk_workspace(be, ca)), dtype=torch.uint8, device="cuda")
    starts, lens = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (bt.q_starts, bt.seq_lens))
    results = []
    for shift in (0, blocks - bt.blocks):
        t = torch.from_numpy(np.where(bt.tables == P.SENTINEL, -1, bt.tables.astype(np.int64) + shift).astype(np.int32)).cuda()
        kp[shift:shift + bt.blocks] = torch.from_numpy(bt.k).cuda().to(dtype)
        vp[shift:shift + bt.blocks] = torch.from_numpy(bt.v).cuda().to(dtype)
        q, out = (torch.zeros(bt.rows, bt.heads * dh, device="cuda") for _ in range(2))
        h = [be.import_tensor(x) for x in (qkv, cos, sin, t, starts, lens, kp, vp, q, out, ws)]
        stream = torch.cuda.current_stream().cuda_stream
        be.wait_stream(stream)
        P.rope_paged_kv_append(be, *h[:8], aa, h[8])
        P.paged_chunk_attention(be, h[8], h[6], h[7], h[3], h[4], h[5], ca, h[10], h[9])
        be.stream_wait(stream)
        results.append([x.clone() for x in (q, out, kp[shift:shift + bt.blocks], vp[shift:shift + bt.blocks])])
        be.synchronize_device()
        for x in h:
            x.release()
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[0][1].abs().sum(1).gt(0).all())
    del kp, vp, results
    torch.cuda.empty_cache()


def test_contexts_side_by_side(be):
    """Two contexts with streams and workspaces of their own: launches of all forms overlap on the GPU and answer as they do alone."""
    other = Backend(0)
    try:
        jobs = []
        for ctx, seed in ((be, 90), (other, 91)):
            for kw, io_bf16 in ((dict(new=[1] * 60, total=[700] * 60), False), (dict(new=[300, 1, 5], total=[900, 2000, 60]), True),
                                (dict(new=[90, 20], total=[400, 1500], dh=64, heads=4, kv_heads=4), False)):
                bt = Batch(seed=seed, **kw)
                q = bf16(bt.q) if io_bf16 else bt.q
                want = run_attention(ctx, bt, q, io_bf16, 0.1)
                args = P.PagedChunkArgs(layout_of(bt), bt.batch, bt.rows, max(bt.new), max(bt.total), bt.heads, bt.kv_heads, bt.width, 0.1,
                                        BF16 if io_bf16 else F32)
                ws = ctx.alloc_zeroed((max(16, P.paged_chunk_workspace(ctx, args)),), np.uint8)
                operands = (up(ctx, q, io_bf16), up(ctx, bt.k, True), up(ctx, bt.v, True), ctx.upload(bt.tables), ctx.upload(bt.q_starts),
                            ctx.upload(bt.seq_lens), args, ws)
                jobs.append((ctx, want, io_bf16, operands, up(ctx, np.zeros_like(q), io_bf16)))
        be.synchronize_device()
        other.synchronize_device()
        for _ in range(20):
            for i in (0, 3, 1, 4, 2, 5):
                ctx, _, _, operands, out = jobs[i]
                P.paged_chunk_attention(ctx, *operands, out)
        for ctx, want, io_bf16, _, out in jobs:
            assert np.array_equal(down(out, want.shape, io_bf16), want)
    finally:
        other.close()
