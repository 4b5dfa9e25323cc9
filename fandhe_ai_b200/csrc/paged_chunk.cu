// A batch of ragged chunks over the paged KV cache: the append of its keys and values with the rotary rotation on the way, and
// the general form of its attention (paged_chunk_tc5.cuh holds the tensor-core form).
//
// Sequence b brings the token rows [q_starts[b], q_starts[b + 1]); it holds seq_lens[b] cached tokens of which those rows are the
// last, so row r of it stands at position seq_lens[b] - (q_starts[b + 1] - r).  All three arrays live on the device; nothing in
// them is trusted: an index out of range sets the error word and touches nothing.
#include <type_traits>

#include "kernels.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace b200 {
namespace {

// What a sequence's entries [s, e) of q_starts and its length must satisfy; nothing is read or written for one that does not.
__device__ __forceinline__ bool sequence_ok(const RaggedShape& sh, uint32_t s, uint32_t e, uint32_t len) {
    return e >= s && e <= static_cast<uint32_t>(sh.rows) && e - s <= len && e - s <= static_cast<uint32_t>(sh.max_q_len) &&
           len <= static_cast<uint32_t>(sh.max_seq_len);
}
// The same for all sequences, by one warp of a launch: the kernels whose blocks look at single rows do not meet every entry.
__device__ __forceinline__ void check_sequences(const RaggedShape& sh, const uint32_t* __restrict__ q_starts,
                                                const uint32_t* __restrict__ seq_lens, uint32_t* err) {
    for (int b = threadIdx.x & 31; b < sh.batch; b += 32)
        if (!sequence_ok(sh, q_starts[b], q_starts[b + 1], seq_lens[b])) atomicCAS(err, 0u, static_cast<uint32_t>(kErrRaggedBatch));
}

// Index of the sequence that row `row` belongs to, by one pass of the whole block over q_starts (one load latency instead of the
// log2(batch) dependent ones of a binary search): the number of starts[1..batch] that are <= row.  `batch` when it belongs to none.
// Only a guess where the starts decrease: the caller asks whether the row stands in [starts[seq], starts[seq + 1]).
__device__ __forceinline__ int sequence_of_row(const uint32_t* __restrict__ q_starts, int batch, int64_t row) {
    int seq = 0;
    for (int b0 = 0; b0 < batch; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        seq += __syncthreads_count(b < batch && int64_t(q_starts[b + 1]) <= row);
    }
    return seq;
}

// ------------------------------------------------------------------------------------ append
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(uint16_t v) { return bf16_bits_to_f32(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float v) {      // round to nearest even
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&x)[N]) {
    constexpr int W = sizeof(T) * N > 16 ? 16 / sizeof(T) : N;      // at most 16 bytes an access
#pragma unroll
    for (int g = 0; g < N; g += W) {
        const Pack<T, W> raw = *reinterpret_cast<const Pack<T, W>*>(p + g);
#pragma unroll
        for (int k = 0; k < W; ++k) x[g + k] = as_f32(raw.v[k]);
    }
}
// ... of what nobody reads again
template <typename T, int N>
__device__ __forceinline__ void load_once(const T* p, float (&x)[N]) {
    if constexpr (sizeof(T) * N == 16) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
        const Pack<T, N> raw = *reinterpret_cast<const Pack<T, N>*>(&u);
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = as_f32(raw.v[k]);
    } else {
        load_f32<T, N>(p, x);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&x)[N]) {
    constexpr int W = sizeof(T) * N > 16 ? 16 / sizeof(T) : N;
#pragma unroll
    for (int g = 0; g < N; g += W) {
        Pack<T, W> raw;
        if constexpr (sizeof(T) == 2 && W % 2 == 0) {
#pragma unroll
            for (int k = 0; k < W; k += 2)
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(reinterpret_cast<uint32_t*>(&raw)[k / 2]) : "f"(x[g + k + 1]), "f"(x[g + k]));
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k) raw.v[k] = from_f32<T>(x[g + k]);
        }
        *reinterpret_cast<Pack<T, W>*>(p + g) = raw;
    }
}

constexpr int kAppendRows = 8;      // at most, token rows of a block
struct AppendRow {
    int64_t slot, angle;            // first element of the token's pool row, row of the cos / sin tables; slot < 0: nothing to do
};

// A block takes `rows_per_block` consecutive token rows (with few rows one, whose heads grid.y blocks share).  Warp r finds out where
// the r-th of them goes, then all threads go through the rows' units of work together.  A unit is a pair of N-element groups that
// rotate into each other (ADJ: one group holding N / 2 pairs) or a group that is copied; N elements are 16 bytes of the activation
// type, or N = 1 (ADJ: 2) where an alignment or a size does not allow that.  Bound by HBM where rows are long: 8192 f32 rows of 24 KB in
// 65.5 us (5.7 TB/s); 14k bf16 rows of 4.6 KB in 41 us (3.6 TB/s); 128 rows in 5.8 us, the launch.
// Eight blocks fit an SM with 32 registers, which the adjacent form has to be told (it chose 31 and took 42.9 us instead of 41.0).
template <typename T, typename KvT, int N, bool ADJ>
__global__ void __launch_bounds__(256, ADJ ? 8 : 0)
rope_append_kernel(RaggedShape sh, RopeShape rope, int rows_per_block, const T* __restrict__ qkv, const float* __restrict__ cos_t,
                   const float* __restrict__ sin_t, const uint32_t* __restrict__ positions, const uint32_t* __restrict__ tables,
                   const uint32_t* __restrict__ q_starts, const uint32_t* __restrict__ seq_lens, T* __restrict__ q_out,
                   KvT* __restrict__ k_pool, KvT* __restrict__ v_pool, uint32_t* err) {
    __shared__ AppendRow place[kAppendRows];
    const int64_t row0 = int64_t(blockIdx.x) * rows_per_block;
    const int count = int(min(int64_t(rows_per_block), sh.rows - row0));
    const int64_t ekv = int64_t(sh.num_kv_heads) * sh.head_dim;
    for (int i = threadIdx.x >> 5; i < count; i += blockDim.x >> 5) {
        const int64_t row = row0 + i;
        const int lane = threadIdx.x & 31;
        int seq = 0;                       // the number of starts[1 .. batch] that are <= row: one load latency, no search
        for (int b0 = 0; b0 < sh.batch; b0 += 128) {
            int before = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int b = b0 + k * 32 + lane;
                before += b < sh.batch && int64_t(q_starts[b + 1]) <= row;
            }
            seq += int(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(before)));
        }
        if (lane == 0) {
            AppendRow to = {-1, 0};
            seq = min(seq, sh.batch - 1);
            const uint32_t from = q_starts[seq], upto = q_starts[seq + 1], len = seq_lens[seq], r = static_cast<uint32_t>(row);
            if (r >= from && r < upto) {                                    // else behind the last sequence
                const uint32_t pos = len - (upto - r);                      // position in the cache
                const uint32_t angle = positions ? positions[row] : pos;
                to.angle = angle;
                if (!sequence_ok(sh, from, upto, len) || (rope.rotary_dim > 0 && angle >= static_cast<uint32_t>(rope.n_positions))) {
                    atomicCAS(err, 0u, static_cast<uint32_t>(kErrRaggedBatch));
                } else {
                    const uint32_t blk = tables[int64_t(seq) * sh.max_blocks_per_seq + pos / static_cast<uint32_t>(sh.block_size)];
                    if (blk >= uint32_t(sh.num_blocks)) atomicCAS(err, 0u, static_cast<uint32_t>(kErrAppendSlot));
                    else to.slot = (int64_t(blk) * sh.block_size + pos % static_cast<uint32_t>(sh.block_size)) * ekv;
                }
            }
            place[i] = to;
        }
    }
    // (the last warp: with one row to a block it has nothing else to do here)
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x + 32 >= blockDim.x) check_sequences(sh, q_starts, seq_lens, err);
    __syncthreads();
    const int d = sh.head_dim, half = rope.rotary_dim / 2;
    const int turned = ADJ ? rope.rotary_dim / N : half / N;            // units of a head that rotate
    const int units = turned + (d - rope.rotary_dim) / N;
    const int turning_heads = sh.num_q_heads + sh.num_kv_heads;
    const int total = turning_heads * units + sh.num_kv_heads * (d / N);
#pragma unroll 1
    for (int w0 = blockIdx.y * blockDim.x + threadIdx.x; w0 < total * count; w0 += gridDim.y * blockDim.x) {
        const int i = w0 / total, w = w0 - i * total;
        const int64_t slot = place[i].slot, row = row0 + i;
        if (slot < 0) continue;
        const T* src = qkv + row * sh.row_stride;
        T* q_row = q_out + row * (int64_t(sh.num_q_heads) * d);
        const float* c_row = cos_t + place[i].angle * half;
        const float* s_row = sin_t + place[i].angle * half;
        if (w >= turning_heads * units) {                               // v: a copy
            const int e = (w - turning_heads * units) * N;
            float x[N];
            load_once<T, N>(src + int64_t(turning_heads) * d + e, x);
            store_f32<KvT, N>(v_pool + slot + e, x);
            continue;
        }
        const int head = w / units, unit = w % units;
        const T* h = src + int64_t(head) * d;
        const bool is_q = head < sh.num_q_heads;
        auto put = [&](int e, const float (&x)[N]) {
            if (is_q) store_f32<T, N>(q_row + int64_t(head) * d + e, x);
            else store_f32<KvT, N>(k_pool + slot + int64_t(head - sh.num_q_heads) * d + e, x);
        };
        if (unit >= turned) {
            const int e = rope.rotary_dim + (unit - turned) * N;
            float x[N];
            load_once<T, N>(h + e, x);
            put(e, x);
        } else if constexpr (ADJ) {
            const int e = unit * N;
            float x[N], c[N / 2], s[N / 2], y[N];
            load_once<T, N>(h + e, x);
            load_f32<float, N / 2>(c_row + e / 2, c);
            load_f32<float, N / 2>(s_row + e / 2, s);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
                y[2 * k] = fmaf(x[2 * k], c[k], -(x[2 * k + 1] * s[k]));
                y[2 * k + 1] = fmaf(x[2 * k + 1], c[k], x[2 * k] * s[k]);
            }
            put(e, y);
        } else {
            const int e = unit * N;
            float a[N], b[N], c[N], s[N], ya[N], yb[N];
            load_once<T, N>(h + e, a);
            load_once<T, N>(h + e + half, b);
            load_f32<float, N>(c_row + e, c);
            load_f32<float, N>(s_row + e, s);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                ya[k] = fmaf(a[k], c[k], -(b[k] * s[k]));
                yb[k] = fmaf(b[k], c[k], a[k] * s[k]);
            }
            put(e, ya);
            put(e + half, yb);
        }
    }
}

template <typename T, typename KvT>
cudaError_t launch_append(const RaggedShape& sh, const RopeShape& rope, const void* qkv, const float* cos_t, const float* sin_t,
                          const uint32_t* positions, const uint32_t* tables, const uint32_t* q_starts, const uint32_t* seq_lens, void* q_out,
                          void* k_pool, void* v_pool, int sm_count, uint32_t* err, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    // 16-byte accesses: every group of N elements starts on such a boundary in all six arrays
    const bool wide = aligned(qkv) && aligned(q_out) && aligned(k_pool) && aligned(v_pool) && aligned(cos_t) && aligned(sin_t) &&
                      sh.row_stride % N == 0 && sh.head_dim % 8 == 0 && rope.rotary_dim % (2 * N) == 0;
    const int per_row = (sh.num_q_heads + 2 * sh.num_kv_heads) * sh.head_dim / (wide ? 2 * N : 2);
    // Many rows: as many to a block as make about 2048 units of work, at most eight (8192 f32 rows of 24 KB: 65.6 us with two rows to a
    // block, 71.3 with eight; 14k bf16 rows of 4.6 KB: 65.5 us with one, 40 with eight).  Few rows: one, shared out over as many
    // blocks as keep every SM busy with 64 units of work each.
    const int wanted = 2048 / (per_row > 0 ? per_row : 1);
    const int per_block = sh.rows < int64_t(4) * kAppendRows * sm_count ? 1 : (wanted < 1 ? 1 : (wanted < kAppendRows ? wanted : kAppendRows));
    int split = 1;
    while (split < 16 && sh.rows * split < 2 * sm_count && per_row / (2 * split) >= 64) split *= 2;
    int threads = 256;
    while (per_block == 1 && threads > 64 && per_row / split <= threads / 2) threads /= 2;
    const dim3 grid(static_cast<unsigned>((sh.rows + per_block - 1) / per_block), split);
#define B200_APPEND(NN, ADJ)                                                                                                             \
    rope_append_kernel<T, KvT, NN, ADJ><<<grid, threads, 0, s>>>(sh, rope, per_block, static_cast<const T*>(qkv), cos_t, sin_t, positions, tables,     \
                                                                 q_starts, seq_lens, static_cast<T*>(q_out), static_cast<KvT*>(k_pool), \
                                                                 static_cast<KvT*>(v_pool), err)
    if (wide) {
        if (rope.adjacent) B200_APPEND(N, true);
        else B200_APPEND(N, false);
    } else if (rope.adjacent && sh.head_dim % 2 == 0 && sh.row_stride % 2 == 0) {
        B200_APPEND(2, true);
    } else {
        B200_APPEND(1, false);
    }
#undef B200_APPEND
    return cudaGetLastError();
}

// ------------------------------------------------------------------------------------ attention, general form
constexpr int kGenThreads = 128;
constexpr int kGenMaxDimsPerLane = 8;   // head_dim <= 256

// One block per (token row, query head): four warps walk the visible keys, each with its own running maximum and sum, lanes stride
// the head; the warps are merged at the end.  Any head_dim up to 256, any block size, f32 or bf16 pools.  A key beyond a row's
// mask is not read, so what stands there does not matter.
template <typename T, typename KvT>
__global__ void __launch_bounds__(kGenThreads)
paged_chunk_generic_kernel(RaggedShape sh, const T* __restrict__ q, const KvT* __restrict__ k_pool, const KvT* __restrict__ v_pool,
                           const uint32_t* __restrict__ tables, const uint32_t* __restrict__ q_starts,
                           const uint32_t* __restrict__ seq_lens, T* __restrict__ out, uint32_t* err) {
    __shared__ float red_m[4], red_l[4];
    __shared__ float red_o[4][256];
    const int64_t row = blockIdx.x;
    const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = sequence_of_row(q_starts, sh.batch, row);
    if (row == 0 && h == 0 && warp == 0) check_sequences(sh, q_starts, seq_lens, err);
    if (seq >= sh.batch) return;
    const int64_t from = q_starts[seq], upto = q_starts[seq + 1], len = seq_lens[seq];
    if (row < from || row >= upto) return;
    const int dh = sh.head_dim;
    const int64_t limit = sequence_ok(sh, from, upto, len) ? len - (upto - row) + 1 : 0;       // visible keys
    const int kvh = h / (sh.num_q_heads / sh.num_kv_heads);
    const int64_t ekv = int64_t(sh.num_kv_heads) * dh;
    const T* q_row = q + row * sh.row_stride + int64_t(h) * dh;
    T* o_row = out + (row * sh.num_q_heads + h) * dh;
    float qs[kGenMaxDimsPerLane], acc[kGenMaxDimsPerLane];
#pragma unroll
    for (int t = 0; t < kGenMaxDimsPerLane; ++t) {
        const int d = lane + 32 * t;
        qs[t] = d < dh ? as_f32(q_row[d]) : 0.0f;
        acc[t] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    bool bad = false;
    for (int64_t j = warp; j < limit; j += 4) {
        const uint32_t blk = tables[int64_t(seq) * sh.max_blocks_per_seq + j / sh.block_size];
        if (blk >= uint32_t(sh.num_blocks)) { bad = true; break; }
        const int64_t off = (int64_t(blk) * sh.block_size + j % sh.block_size) * ekv + int64_t(kvh) * dh;
        float s = 0.0f;
#pragma unroll
        for (int t = 0; t < kGenMaxDimsPerLane; ++t) {
            const int d = lane + 32 * t;
            if (d < dh) s = fmaf(qs[t], as_f32(k_pool[off + d]), s);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= sh.scale;
        const float m_new = m > s || m != m ? m : s;      // NaN stays
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = expf(m - base), p = expf(s - base);
        l = fmaf(l, corr, p);
#pragma unroll
        for (int t = 0; t < kGenMaxDimsPerLane; ++t) {
            const int d = lane + 32 * t;
            if (d < dh) acc[t] = fmaf(p, as_f32(v_pool[off + d]), acc[t] * corr);
        }
        m = m_new;
    }
    if (lane == 0) { red_m[warp] = m; red_l[warp] = l; }
#pragma unroll
    for (int t = 0; t < kGenMaxDimsPerLane; ++t) {
        const int d = lane + 32 * t;
        if (d < dh) red_o[warp][d] = acc[t];
    }
    const int any_bad = __syncthreads_or(bad ? 1 : 0);
    if (any_bad) {
        if (threadIdx.x == 0) atomicCAS(err, 0u, static_cast<uint32_t>(kErrAttnBlockId));
        for (int d = threadIdx.x; d < dh; d += kGenThreads) o_row[d] = from_f32<T>(__int_as_float(0x7FC00000));
        return;
    }
    float w[4], ll = 0.0f, mm = red_m[0];
#pragma unroll
    for (int t = 1; t < 4; ++t) mm = mm > red_m[t] || mm != mm ? mm : red_m[t];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        w[t] = red_m[t] == -INFINITY ? 0.0f : expf(red_m[t] - mm);
        ll = fmaf(red_l[t], w[t], ll);
    }
    for (int d = threadIdx.x; d < dh; d += kGenThreads) {
        float o = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) o = fmaf(red_o[t][d], w[t], o);
        if (o != o && ll > 0.0f && ll < INFINITY) {      // infinities that met weights of zero, or NaN: the values themselves
            float extra = 0.0f;
            for (int64_t j = 0; j < limit; ++j) {
                const int64_t blk = tables[int64_t(seq) * sh.max_blocks_per_seq + j / sh.block_size];
                const float v = as_f32(v_pool[(blk * sh.block_size + j % sh.block_size) * ekv + int64_t(kvh) * dh + d]);
                if (!(fabsf(v) < INFINITY)) extra += v;
            }
            if (extra != 0.0f) o = extra;
        }
        o_row[d] = from_f32<T>(limit > 0 ? o / ll : 0.0f);
    }
}

#include "paged_chunk_tc5.cuh"

// What a call launches: decided from the arguments alone, so that the workspace query and the call agree.
struct ChunkPlan {
    bool tc5;
    int64_t items;             // upper bound
    int chunk_tiles, max_chunks;
};

constexpr int kFewRows = 10;      // TcCfg<., true>::kTinyRows

ChunkPlan plan_chunk(const RaggedShape& sh, int io_bf16, int kv_bf16, int sm_count) {
    ChunkPlan plan = {false, 0, 0, 1};
    const int item = io_bf16 ? 2 : 4;
    if (!kv_bf16 || (sh.head_dim != 64 && sh.head_dim != 128) || sh.block_size < 8 || (sh.row_stride * item) % 16 != 0 ||
        int64_t(sh.num_blocks) * sh.block_size > 0x7FFFFFFF || sh.max_seq_len == 0)
        return plan;
    const int64_t group = sh.num_q_heads / sh.num_kv_heads, rows = io_bf16 ? 256 : 128;
    const int64_t by_len = int64_t(sh.batch) * ((int64_t(sh.max_q_len) * group + rows - 1) / rows);
    const int64_t by_rows = sh.rows * group / rows + (sh.rows < sh.batch ? sh.rows : sh.batch);
    const int64_t units = (by_len < by_rows ? by_len : by_rows) * sh.num_kv_heads;
    const int tiles = (sh.max_seq_len + kTcKeys - 1) / kTcKeys;
    // Key ranges per row: the number that makes the launch shortest when an item costs its key tiles plus about three tiles of
    // start and finish, and the items are dealt out to the SMs in equal rounds.  The variant for few f32 rows has ranges of at most
    // 6144 keys: its accumulators are cut at every addition (see the kernel), and nothing is put aside there.
    const int longest = !io_bf16 && int64_t(sh.max_q_len) * group <= kFewRows ? 48 : tiles;
    int best = 1, best_over = INT32_MAX;      // over: tiles beyond the longest range
    int64_t best_cost = INT64_MAX;
    for (int n = 1; n <= 64 && (n == 1 || tiles / n >= 2); ++n) {
        const int per = (tiles + n - 1) / n, count = (tiles + per - 1) / per, over = per > longest ? per - longest : 0;
        if (count > 1 && sh.rows * sh.num_q_heads * count * (sh.head_dim * 4 + 8) > (int64_t(512) << 20)) break;
        const int64_t cost = ((units * count + sm_count - 1) / sm_count) * (per + 3);
        if (over < best_over || (over == best_over && cost < best_cost)) {
            best_over = over;
            best_cost = cost;
            best = n;
        }
    }
    plan.chunk_tiles = (tiles + best - 1) / best;
    plan.max_chunks = (tiles + plan.chunk_tiles - 1) / plan.chunk_tiles;
    plan.items = units * plan.max_chunks;
    // (32 sequences of any length within the bounds, whatever q_starts holds: a warp adds their items up in 32 bits)
    const int64_t of_32 = 32 * ((int64_t(sh.max_q_len) * group + rows - 1) / rows) * sh.num_kv_heads * plan.max_chunks;
    plan.tc5 = plan.items < 0x7FFFFFFF && of_32 < 0x7FFFFFFF && int64_t(sh.max_q_len) * group < 0x7FFFFFFF;
    return plan;
}

static_assert(TcCfg<64, true>::kTinyRows == kFewRows && TcCfg<128, true>::kTinyRows == kFewRows, "");

template <int D, bool F32, bool TINY, typename T>
cudaError_t launch_tc5_kind(const ChunkPlan& plan, const RaggedShape& sh, const void* q, const void* k_pool, const void* v_pool,
                       const uint32_t* tables, const uint32_t* q_starts, const uint32_t* seq_lens, void* workspace, void* out, int sm_count,
                       uint32_t* err, cudaStream_t s) {
    using Cfg = TcCfg<D, F32>;
    static int configured[64] = {};
    if (cudaError_t e = ensure_dynamic_smem(paged_chunk_tc5_kernel<D, F32, TINY, T>, Cfg::kSmem, configured)) return e;
    CUtensorMap map_k, map_v;
    const int64_t pool_rows = int64_t(sh.num_blocks) * sh.block_size, ekv = int64_t(sh.num_kv_heads) * D;
    const int box = sh.block_size < kTcKeys ? sh.block_size : kTcKeys;
    if (!make_bf16_rows_map(&map_k, k_pool, pool_rows, ekv, 64, box) || !make_bf16_rows_map(&map_v, v_pool, pool_rows, ekv, 64, box))
        return cudaErrorInvalidValue;
    TcShape p;
    p.sh = sh;
    p.group = sh.num_q_heads / sh.num_kv_heads;
    p.chunk_tiles = plan.chunk_tiles;
    p.max_chunks = plan.max_chunks;
    p.q_sign = sh.scale < 0.0f ? -1.0f : 1.0f;
    // scale 0: a factor so small that every finite score gives a weight of one, and a masked one (-inf) still none
    p.scale_log2 = fmaxf(fabsf(sh.scale) * 1.44269504088896341f, 1.2e-38f);
    float* part_o = static_cast<float*>(workspace);
    float2* part_ml = reinterpret_cast<float2*>(part_o + (plan.max_chunks > 1 ? sh.rows * sh.num_q_heads * plan.max_chunks * D : 0));
    const dim3 grid(static_cast<unsigned>(plan.items));
    cudaError_t e = launch_ex(paged_chunk_tc5_kernel<D, F32, TINY, T>, grid, dim3(kTcThreads), Cfg::kSmem, s, 1, true, map_k, map_v, p,
                              static_cast<const T*>(q), static_cast<const uint16_t*>(k_pool), static_cast<const uint16_t*>(v_pool), tables, q_starts, seq_lens,
                              static_cast<T*>(out), part_o, part_ml, err);
    if (e != cudaSuccess || plan.max_chunks == 1) return e;
    const dim3 join(static_cast<unsigned>(sh.rows), (sh.num_q_heads + 7) / 8);
    return launch_ex(paged_chunk_join_kernel<D, T>, join, dim3(256), 0, s, 1, true, p, Cfg::kRows, q_starts, seq_lens, part_o, part_ml,
                     static_cast<T*>(out));
}

template <int D, bool F32, typename T, typename... Args>
cudaError_t launch_tc5(const ChunkPlan& plan, const RaggedShape& sh, Args... args) {
    if (int64_t(sh.max_q_len) * (sh.num_q_heads / sh.num_kv_heads) <= TcCfg<D, F32>::kTinyRows) return launch_tc5_kind<D, F32, true, T>(plan, sh, args...);
    return launch_tc5_kind<D, F32, false, T>(plan, sh, args...);
}

}  // namespace

cudaError_t rope_paged_kv_append(const RaggedShape& sh, const RopeShape& rope, const void* qkv, int io_bf16, const float* cos_t,
                                 const float* sin_t, const uint32_t* positions, const uint32_t* tables, const uint32_t* q_starts,
                                 const uint32_t* seq_lens, void* q_out, void* k_pool, void* v_pool, int kv_bf16, int sm_count,
                                 uint32_t* err, cudaStream_t s) {
    if (sh.rows == 0 || sh.batch == 0) return cudaSuccess;
    if (io_bf16)
        return kv_bf16 ? launch_append<uint16_t, uint16_t>(sh, rope, qkv, cos_t, sin_t, positions, tables, q_starts, seq_lens, q_out, k_pool, v_pool, sm_count, err, s)
                       : launch_append<uint16_t, float>(sh, rope, qkv, cos_t, sin_t, positions, tables, q_starts, seq_lens, q_out, k_pool, v_pool, sm_count, err, s);
    return kv_bf16 ? launch_append<float, uint16_t>(sh, rope, qkv, cos_t, sin_t, positions, tables, q_starts, seq_lens, q_out, k_pool, v_pool, sm_count, err, s)
                   : launch_append<float, float>(sh, rope, qkv, cos_t, sin_t, positions, tables, q_starts, seq_lens, q_out, k_pool, v_pool, sm_count, err, s);
}

size_t paged_chunk_workspace_bytes(const RaggedShape& sh, int io_bf16, int kv_bf16, int sm_count) {
    const ChunkPlan plan = plan_chunk(sh, io_bf16, kv_bf16, sm_count);
    return plan.tc5 && plan.max_chunks > 1 ? size_t(sh.rows) * sh.num_q_heads * plan.max_chunks * (sh.head_dim * 4 + 8) : 0;
}

cudaError_t paged_chunk_attention(const RaggedShape& sh, const void* q, int io_bf16, const void* k_pool, const void* v_pool, int kv_bf16,
                                  const uint32_t* tables, const uint32_t* q_starts, const uint32_t* seq_lens, void* workspace, void* out,
                                  int sm_count, uint32_t* err, cudaStream_t s) {
    if (sh.rows == 0 || sh.batch == 0) return cudaSuccess;
    const ChunkPlan plan = plan_chunk(sh, io_bf16, kv_bf16, sm_count);
    if (plan.tc5) {
        if (sh.head_dim == 128)
            return io_bf16 ? launch_tc5<128, false, uint16_t>(plan, sh, q, k_pool, v_pool, tables, q_starts, seq_lens, workspace, out, sm_count, err, s)
                           : launch_tc5<128, true, float>(plan, sh, q, k_pool, v_pool, tables, q_starts, seq_lens, workspace, out, sm_count, err, s);
        return io_bf16 ? launch_tc5<64, false, uint16_t>(plan, sh, q, k_pool, v_pool, tables, q_starts, seq_lens, workspace, out, sm_count, err, s)
                       : launch_tc5<64, true, float>(plan, sh, q, k_pool, v_pool, tables, q_starts, seq_lens, workspace, out, sm_count, err, s);
    }
    const dim3 grid(static_cast<unsigned>(sh.rows), sh.num_q_heads);
    auto go = [&](auto t, auto kv) {
        using T = decltype(t);
        using KvT = decltype(kv);
        paged_chunk_generic_kernel<T, KvT><<<grid, kGenThreads, 0, s>>>(sh, static_cast<const T*>(q), static_cast<const KvT*>(k_pool),
                                                                       static_cast<const KvT*>(v_pool), tables, q_starts, seq_lens,
                                                                       static_cast<T*>(out), err);
    };
    if (io_bf16) { if (kv_bf16) go(uint16_t(), uint16_t()); else go(uint16_t(), 0.0f); }
    else { if (kv_bf16) go(0.0f, uint16_t()); else go(0.0f, 0.0f); }
    return cudaGetLastError();
}

}  // namespace b200
