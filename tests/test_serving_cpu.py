"""Serving operators of a ragged batch without a GPU: argument rules, the host validators, the rotary table, and the plain
forms that the GPU tests compare with, checked against hand-made values."""
import math

import numpy as np
import pytest

from fandhe_ai_b200 import BF16, F32, I8, BackendError
from fandhe_ai_b200 import paged_kv as P
from fandhe_ai_b200.decoder import SampleArgs, validate_sample

from serving_ref import Batch, append_ref, attention_ref, sample_ref


def chunk_args(**kw):
    d = dict(layout=P.PagedKvLayout(8, 16, 256, BF16), batch=2, rows=10, max_q_len=8, max_seq_len=48, num_heads=8, num_kv_heads=2,
             max_blocks_per_seq=3, scale=0.1)
    d.update(kw)
    return P.PagedChunkArgs(**d)


TABLES = np.array([[0, 1, 2], [3, 4, P.SENTINEL]], np.uint32)


def test_valid_batches_pass():
    P.validate_ragged_batch(TABLES, [0, 8, 10], [48, 17], chunk_args())
    P.validate_ragged_batch(TABLES, [0, 0, 10], [0, 17], chunk_args(max_q_len=10))            # a sequence without new tokens
    P.validate_ragged_batch(np.zeros((0, 3), np.uint32), [0], [], chunk_args(batch=0, rows=0))
    P.validate_rope_append(P.RopeAppendArgs(P.PagedKvLayout(8, 16, 256, BF16), 2, 10, 8, 2, 3, 128, 48))
    validate_sample(SampleArgs(4, 1000))


@pytest.mark.parametrize("starts,lens,kw,what", [
    ([1, 8, 10], [48, 17], {}, "q_starts[0]"),
    ([0, 8, 7], [48, 17], {}, "decreases"),
    ([0, 9, 10], [48, 17], {}, "max_q_len"),
    ([0, 8, 10], [49, 17], {}, "max_seq_len"),
    ([0, 8, 10], [7, 17], {}, "new tokens, but only"),
    ([0, 8, 10], [48, 33], {}, "block id"),                     # the third block of sequence 1 is the sentinel
    ([0, 8, 10], [48, 17], dict(rows=9), "behind the last row"),
    ([0, 8, 10], [48, 17], dict(layout=P.PagedKvLayout(4, 16, 256, BF16)), "block id 4"),
])
def test_bad_batches_are_refused(starts, lens, kw, what):
    with pytest.raises(BackendError) as e:
        P.validate_ragged_batch(TABLES, starts, lens, chunk_args(**kw))
    assert e.value.kind == "InvalidArgument" and what in e.value.message


@pytest.mark.parametrize("kw,kind", [
    (dict(num_kv_heads=0), "InvalidArgument"),
    (dict(num_kv_heads=3), "InvalidArgument"),
    (dict(num_heads=7), "InvalidArgument"),
    (dict(num_heads=0), "InvalidArgument"),
    (dict(scale=math.inf), "InvalidArgument"),
    (dict(scale=math.nan), "InvalidArgument"),
    (dict(io_dtype=I8), "InvalidArgument"),
    (dict(max_seq_len=49), "InvalidArgument"),
    (dict(max_q_len=49), "InvalidArgument"),
    (dict(q_stride=1023), "InvalidArgument"),
    (dict(rows=1 << 31), "InvalidArgument"),
    (dict(batch=1 << 31), "InvalidArgument"),
    (dict(max_blocks_per_seq=1 << 28), "InvalidArgument"),
    (dict(q_stride=1 << 60), "InvalidArgument"),
    (dict(layout=P.PagedKvLayout(8, 24, 256, BF16)), "InvalidArgument"),
    (dict(layout=P.PagedKvLayout(0, 16, 256, BF16)), "InvalidArgument"),
    (dict(layout=P.PagedKvLayout(8, 16, 256, I8)), "InvalidArgument"),
    (dict(layout=P.PagedKvLayout(1 << 62, 16, 256, BF16)), "InvalidArgument"),
    (dict(layout=P.PagedKvLayout(1 << 31, 16, 256, BF16)), "Unsupported"),
    (dict(layout=P.PagedKvLayout(8, 16, 1024, BF16)), "Unsupported"),       # head_dim 512
    (dict(num_heads=65536 * 2), "Unsupported"),
])
def test_bad_chunk_arguments_are_refused(kw, kind):
    a = chunk_args(**kw)
    with pytest.raises(BackendError) as e:
        P.check(P.lib().b200_validate_ragged_batch(None, None, None, a._c))
    assert e.value.kind == kind


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=130), dict(qkv_stride=12), dict(io_dtype=I8), dict(n_positions=1 << 31),
                                dict(adjacent_pairs=True, qkv_stride=1537), dict(num_heads=5), dict(rows=1 << 32)])
def test_bad_append_arguments_are_refused(kw):
    d = dict(layout=P.PagedKvLayout(8, 16, 256, BF16), batch=2, rows=10, num_heads=8, num_kv_heads=2, max_blocks_per_seq=3, rotary_dim=128,
             n_positions=48)
    d.update(kw)
    with pytest.raises(BackendError) as e:
        P.validate_rope_append(P.RopeAppendArgs(**d))
    assert e.value.kind == "InvalidArgument"


@pytest.mark.parametrize("a,kind", [(SampleArgs(1, 0), "InvalidArgument"), (SampleArgs(1, 393217), "Unsupported"),
                                    (SampleArgs(2, 100, 99), "InvalidArgument"), (SampleArgs(2, 100, dtype=I8), "InvalidArgument"),
                                    (SampleArgs(1 << 40, 100), "InvalidArgument"), (SampleArgs(1 << 20, 100, 1 << 50), "InvalidArgument")])
def test_bad_sample_arguments_are_refused(a, kind):
    with pytest.raises(BackendError) as e:
        validate_sample(a)
    assert e.value.kind == kind


def test_calls_without_a_context_are_refused():
    lib = P.lib()
    for st in (lib.b200_sample_tokens(None, None, 0, SampleArgs(1, 8)._c, *[None] * 8),
               lib.b200_paged_chunk_attention(None, None, 0, None, None, None, None, None, chunk_args()._c, None, None, 0),
               lib.b200_paged_chunk_workspace(None, chunk_args()._c, None), lib.b200_buf_import(None, None, 0, None),
               lib.b200_ctx_wait_stream(None, None), lib.b200_stream_wait_ctx(None, None)):
        assert lib.b200_status_name(st) == b"InvalidArgument"


def test_rope_table_is_the_f64_table_rounded_once():
    cos, sin = P.rope_table(10000.0, 64, 3000)
    p, i = np.arange(3000.0)[:, None], np.arange(32.0)[None]
    ang = p * 10000.0 ** (-2.0 * i / 64)
    # f64 angles differ by their own rounding (2^-53 of up to 3000), far below a half step of f32
    assert np.abs(cos - np.cos(ang)).max() <= 2.0 ** -24 * 1.001 and np.abs(sin - np.sin(ang)).max() <= 2.0 ** -24 * 1.001
    for bad in ((0.0, 64, 4), (math.inf, 64, 4), (1e4, 63, 4), (1e4, 0, 4)):
        with pytest.raises(BackendError):
            P.rope_table(*bad)


def test_reference_attention_on_hand_made_values():
    bt = Batch([2], [3], heads=1, kv_heads=1, dh=2, block=2)
    blk, off = bt.places(0)
    bt.k[blk, off] = [[0, 0], [0, 0], [0, 0]]
    bt.v[blk, off] = [[1, 10], [3, 30], [8, 80]]
    out, _ = attention_ref(bt, np.zeros((2, 2), np.float32), 1.0)
    assert np.allclose(out, [[2, 20], [4, 40]])
    # a mask one key too wide would move the first row: the comparison sees it
    assert not np.allclose(out[0], [4, 40])


def test_reference_append_turns_by_the_angle():
    bt = Batch([1], [1], heads=1, kv_heads=1, dh=4, block=1, spare_blocks=0)
    cos, sin = np.array([[0.0, 1.0]], np.float32), np.array([[1.0, 0.0]], np.float32)      # a quarter turn, no turn
    x = np.array([[1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12]], np.float32)
    (q, k, v), _ = append_ref(bt, x, cos, sin, 4, False)
    assert q.tolist() == [[-3, 2, 1, 4]] and k.ravel().tolist() == [-7, 6, 5, 8] and v.ravel().tolist() == [9, 10, 11, 12]
    (q, _, _), _ = append_ref(bt, x, cos, sin, 4, True)
    assert q.tolist() == [[-2, 1, 3, 4]]


def test_reference_sampling_on_hand_made_rows():
    x = np.log(np.array([4.0, 1.0, 4.0, 1.0]))
    assert sample_ref(x, 1, 0, 1, 0, 0.0)[::2] == (0, 4)
    assert [sample_ref(x, 1, 0, 1, 0, u)[0] for u in (0.39, 0.41, 0.49, 0.51, 0.89, 0.91)] == [0, 1, 1, 2, 2, 3]
    assert sample_ref(x, 1, 3, 1, 0, 0.95)[::2] == (2, 3)          # the tie at the border goes to the lower index
    assert sample_ref(x, 1, 0, 0.45, 0, 0.95)[::2] == (2, 2)
    assert sample_ref(x, 1, 0, 1, 0.5, 0.95)[::2] == (2, 2)
    assert sample_ref(x, 0, 0, 1, 0, 0.95)[:3] == (0, 1.0, 1)
    assert sample_ref([-np.inf] * 3, 1, 0, 1, 0, 0.5)[0] == -1 and sample_ref([0, np.nan], 1, 0, 1, 0, 0.5)[0] == -1
