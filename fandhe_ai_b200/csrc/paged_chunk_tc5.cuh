// Attention of a batch of ragged chunks on the tensor cores (included by paged_chunk.cu): bf16 pools, head_dim 64 or 128, blocks of
// 8 tokens or more.
//
// The query rows of a sequence that share a KV head - G = Hq / Hkv heads of each new token - are one list of rows r = i G + g, so
// that a tile of 128 accumulator rows is full however few tokens a sequence brings and every K / V tile is fetched once for
// all of them.  A work item is (sequence, KV head, tile of rows, range of key tiles of 128 keys); it runs on two accumulator
// slots, each with its own group of four softmax warps (thread = row, so row maxima and sums need no exchange):
//   - rows > 128: slot s holds rows [128 s, 128 s + 128) and both slots use every key tile;
//   - rows <= 128, or f32 activations: both slots hold the same rows and share the key tiles (even / odd); their
//     partial results are joined at the end.
// While one slot is in its softmax, the tensor cores work for the other one.
//
//   S = Q K^T   tcgen05.mma, operands from shared memory (128-byte swizzle, K-major), 128 columns of tensor memory a slot
//   P = 2^(S c - m c), c = scale log2 e; bf16, written over S (the MMA takes both operands in one type, and V is bf16; the sum l is of the
//       f32 weights, so a result is off by the mean of their roundings, 2^-8 each at most, beside the rounding of its own)
//   O += P V    tcgen05.mma, P from tensor memory, V from shared memory as it stands in the cache (MN-major), f32 accumulator
// The running maximum m of a row is raised only when a new score exceeds it by more than 2^8 in the weight: until then the
// weights are merely larger than one, and O need not be rescaled.
//
// f32 activations: q = q1 + q2 + q3 and p = p1 + p2 + p3 as bf16 terms, exact to 24 bits; K and V are bf16, so the products are
// exact and the accumulators f32.  Three times the tensor work; but an item of at most 32 rows ("stacked") has its queries
// three times in the tile of accumulator rows, so that three warps of a group hold the same scores, and each contributes one term
// of the weights: one product gives the three partial results, which are added at the end.
//
// Items of very few rows ("tiny": at most 32, with three terms 10 - single tokens and short drafts) have them in each quarter of the
// tile, term by term: warp w of a group exponentiates the keys [32 w, 32 w + 32) only and leaves its weights of the others at zero, so
// a tile takes a quarter of the time; with three terms a score is put together by shuffles from the partial scores that lanes
// r, r + 10 and r + 20 hold, which takes one product instead of three.  Each warp has its own maximum and sum.  A batch of nothing
// but such items runs in a kernel of its own (TINY): what the other items need would only crowd its instruction cache, and the
// other way round (in one kernel with it, fresh prompts took 270 us instead of 239).
//
// The softmax weights go to the MMA warp in two parts, so that the second product starts while the rest is still in the
// exponential: 96 and 32 keys (little is left to multiply after the last weight), or with three terms 64 and 64.
//
// Warps: 0-7 softmax (two groups); 8 deals out the items (decoded once, into shared memory) and fetches their tiles by TMA (one
// box per cache block and half head, through the block table); 9 and 10 issue the products of one slot each, which keeps the
// chain scores -> softmax -> values of a slot free of the other slot's waits; 11 cleans V: an MMA multiplies what it must not
// see by zero, which does not remove NaN and infinities.  In tiles with
// masked keys (only the last ones of a sequence; such a tile is announced to warp 11, and by it to the MMA warps) rows beyond the item's last visible key are zeroed, non-finite elements
// of rows that some query must not see are replaced by zero, and if there were any the epilogue adds them back to the rows that do see them
// (as it does where a visible infinity met a weight of zero in some term or quarter).
//
// Measured on a B200 (us; 32 / 8 heads of 128 unless said otherwise): 2039 bf16 tokens over 30011 cached ones 1185 to 1225 (the
// power cap decides), which is 846 to 875 TFLOP/s; four prompts of 2048 187 to 198 (694 to 735 TFLOP/s); one f32 token of each of 128
// sequences over 256 to 2048 184 (3.2 TB/s); four chunks of about 400 f32 tokens among 60 single ones 266; sixteen f32 prompts of 300 to
// 1024, 12 heads of 64, 162; four drafted bf16 tokens of eight sequences 21.  Bound by the chain of a slot and, for short
// items, by their start and finish; not by HBM and not by the tensor cores' rate: the long case takes 2.8 us a key tile and SM,
// both slots together, which is 4700 clocks at its 1690 MHz, where the products of both take 2048 and their exponentials 2048.
// What an item does once is kept short for that reason (prompts, step by step): code that runs once is not
// unrolled, since the instruction cache shows (239 -> 213); bf16 queries go to shared memory by asynchronous copies (213 -> 196);
// finished bf16 rows leave in one pass, staged as bf16 (196 -> 188 in that run).

constexpr int kTcSoftmaxWarps = 8;
// Registers a thread: 168 at launch (384 threads); the softmax threads hold a row of 128 scores and take 216, the other four warps
// give theirs up: 256 x 216 + 128 x 72 = 384 x 168.
constexpr int kTcThreads = 32 * (kTcSoftmaxWarps + 4);
constexpr int kTcKeys = 128;               // keys of a tile
constexpr int kTcBookBytes = 3 << 10;      // of shared memory, for everything but tiles
constexpr int kTcItemSlots = 4;            // items known ahead

template <int D, bool F32>
struct TcCfg {
    static constexpr int kQTerms = F32 ? 3 : 1;
    static constexpr int kPTerms = F32 ? 3 : 1;
    static constexpr int kTileBytes = kTcKeys * D * 2;                       // a K or V tile
    static constexpr int kQTileBytes = 128 * D * 2;
    static constexpr int kQBytes = (F32 ? 3 : 2) * kQTileBytes;              // also holds what the groups exchange at the end of an item
    static constexpr int kStages = D == 128 ? (F32 ? 4 : 5) : 8;
    static constexpr int kSmem = kQBytes + kStages * kTileBytes + kTcBookBytes;
    static constexpr int kRows = F32 ? 128 : 256;                            // rows of an item
    static constexpr int kTinyRows = F32 ? 10 : 32;
    static constexpr int kHold = 2, kHoldStack = 6;                          // f32: tiles of a slot after which O is put aside
};

struct TcShape {
    RaggedShape sh;
    int group, chunk_tiles, max_chunks;
    float scale_log2;          // > 0
    float q_sign;              // -1 for a negative scale: the queries are negated (f32: as they are split; bf16: by the MMA)
};

struct TcItem {
    int seq, kvh, row0, rows, chunk, nchunks;      // row0: first row of the tile in the sequence's list of rows
    int t0, nt;                                    // key tiles [t0, t0 + nt)
    int n, len, start;                             // new tokens, cached tokens, first token row
    int min_limit, max_limit;                      // visible keys of the first and the last row
    bool split, stack;                             // the slots share the rows; the three terms share the accumulator rows
    uint32_t nonfinite;                            // set when cleaning met non-finite values
};

// Walks the items of a launch in increasing order; all lanes of a warp together.
template <int R, bool F32>
struct TcWalk {
    const TcShape& p;
    const uint32_t* q_starts;
    const uint32_t* seq_lens;
    int lane, first = -32, total = 0, incl = 0, items = 0, n = 0, len = 0, start = 0;
    int64_t base = 0;

    __device__ TcWalk(const TcShape& p_, const uint32_t* a, const uint32_t* b) : p(p_), q_starts(a), seq_lens(b), lane(threadIdx.x & 31) {}

    __device__ __forceinline__ int tiles_of_rows() const { return (n * p.group + R - 1) / R; }
    __device__ __forceinline__ int chunks_of_len() const { return ((len + kTcKeys - 1) / kTcKeys + p.chunk_tiles - 1) / p.chunk_tiles; }

    __device__ bool next_group(uint32_t* err) {
        base += total;
        total = 0;
        if (first >= p.sh.batch) return false;
        first += 32;
        if (first >= p.sh.batch) return false;
        const int b = first + lane;
        items = n = len = 0;
        if (b < p.sh.batch) {
            const int64_t s = q_starts[b], e = q_starts[b + 1], l = seq_lens[b];
            if (!sequence_ok(p.sh, s, e, l)) {
                if (err) atomicCAS(err, 0u, static_cast<uint32_t>(kErrRaggedBatch));
            } else if (e > s) {
                n = int(e - s);
                len = int(l);
                start = int(s);
                items = tiles_of_rows() * chunks_of_len() * p.sh.num_kv_heads;
            }
        }
        incl = items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        total = __shfl_sync(0xffffffffu, incl, 31);
        return true;
    }
    // the item `index` (quickest when not below the last one asked for); false when there are no more.  nt = 0: nothing to do.
    __device__ bool get(int64_t index, TcItem& it, uint32_t* err) {
        if (index < base) {
            first = -32;
            base = total = 0;
        }
        while (index >= base + total)
            if (!next_group(err)) return false;
        const int local = int(index - base);
        const uint32_t m = __ballot_sync(0xffffffffu, incl > local);
        const int src = __ffs(m) - 1;
        const int within = local - (__shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, items, src));
        it.seq = first + src;
        it.n = __shfl_sync(0xffffffffu, n, src);
        it.len = __shfl_sync(0xffffffffu, len, src);
        it.start = __shfl_sync(0xffffffffu, start, src);
        const int rows_all = it.n * p.group;
        const int nq = (rows_all + R - 1) / R;
        it.nchunks = ((it.len + kTcKeys - 1) / kTcKeys + p.chunk_tiles - 1) / p.chunk_tiles;
        it.kvh = within % p.sh.num_kv_heads;
        const int rest = within / p.sh.num_kv_heads;
        it.chunk = rest % it.nchunks;
        const int qt = nq - 1 - rest / it.nchunks;              // the tiles that see most keys first
        it.row0 = qt * R;
        it.rows = min(R, rows_all - it.row0);
        it.min_limit = it.len - it.n + it.row0 / p.group + 1;
        it.max_limit = it.len - it.n + (it.row0 + it.rows - 1) / p.group + 1;
        const int tiles = (it.max_limit + kTcKeys - 1) / kTcKeys;
        it.t0 = it.chunk * p.chunk_tiles;
        it.nt = max(0, min(tiles, it.t0 + p.chunk_tiles) - it.t0);
        it.split = F32 || it.rows <= 128;
        it.stack = F32 && it.rows <= 32;
        it.nonfinite = 0;
        return true;
    }
};

// Places of the tiles in the ring: K tiles run `ahead` tiles ahead of the V tiles (1, or 2 when the slots take turns).
struct TcOrder {
    uint32_t p0;
    int n, ahead;
    __device__ __forceinline__ TcOrder(uint32_t p0_, const TcItem& it) : p0(p0_), n(it.nt), ahead(min(it.split ? 2 : 1, it.nt)) {}
    __device__ __forceinline__ uint32_t k(int t) const { return t < ahead ? p0 + t : p0 + 2 * t - ahead + 1; }
    __device__ __forceinline__ uint32_t v(int t) const { return t < n - ahead ? p0 + ahead + 2 * t : p0 + n + t; }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 -> packed bf16, the first in the low half
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

__device__ __forceinline__ float max_nan(float a, float b) {       // NaN if one of them is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t max_nan_bf16(uint32_t a, uint32_t b) {      // of two bf16 each; 0x7FFF where one is NaN
    uint32_t y;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// Two f32 operations in one instruction
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

// Shared-memory descriptor of an MN-major operand whose rows (one per K index) are 128 bytes of the M / N dimension, 128-byte
// swizzled: 8-row groups along K are 1024 bytes apart, the next 64 elements along M / N start `lead` bytes further.
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t smem_addr, uint32_t lead) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(lead >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
__device__ __forceinline__ void umma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_bf16_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld_32x1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
    return r;
}
__device__ __forceinline__ void tmem_st_32x1(uint32_t taddr, uint32_t r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 16 bytes from global to shared memory without a register in between; zeros where `real` is false
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Asks the launch unit for a block of this grid that has not started: that block is cancelled and its work is the caller's.  The
// answer (16 bytes) arrives on the barrier.  Not to be asked again once the answer was "none".
__device__ __forceinline__ void steal_block(uint32_t answer, uint32_t bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int stolen_block(uint32_t answer) {      // -1: none
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred P;\n\t.reg .b128 A;\n\t"
        "ld.shared.b128 A, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 P, A;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@P clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, A;\n\t}\n"
        : "=r"(ok), "=r"(x)
        : "r"(answer)
        : "memory");
    return ok ? static_cast<int>(x) : -1;
}

// First column, counted from a slot's scores, of the bf16 weights of half `h` and term `term` (one term: columns 0 to 63).  Three terms of 64 keys take 96 of the
// 128 columns; the second half's last two terms go to columns that a 64-wide accumulator leaves free, or with D = 128 over the first
// half's once that has been multiplied (p_free).
template <int D>
__device__ __forceinline__ constexpr uint32_t weight_columns(int h, int term) {
    if (h == 0) return term * 32;
    return term == 0 ? 96 : (D == 64 ? 256 + 64 : 0) + (term - 1) * 32;
}
// Two f32 in truncated bf16 (their upper halves), the first in the low half; the remainders are exact
__device__ __forceinline__ uint32_t cut_bf16(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
__device__ __forceinline__ F2 cut_rest(float lo, float hi) {
    return fma2(F2(__uint_as_float(__float_as_uint(lo) & 0xFFFF0000u), __uint_as_float(__float_as_uint(hi) & 0xFFFF0000u)), F2(-1.0f, -1.0f), F2(lo, hi));
}

struct TcShared {
    // Two `full` barriers a stage, taken in turn: a slot that shares the key tiles waits for its own only, so it may ask for a stage
    // while the other slot's tile before it has not landed - with one barrier, whose phase before that is complete, the wait would pass.
    uint64_t full[2][8], empty[8], raw[8];     // raw: a V tile with masked keys has landed and is to be cleaned
    uint64_t s_full[2], p_full[2][2], p_free[2], o_full[2], q_full[2];
    uint32_t turn[4];                          // taken by one of the two softmax warps of a scheduler
    uint64_t meet_all, meet[2];                // the softmax warps meet: all of them, one group
    uint32_t tmem;
    uint64_t item_full[kTcItemSlots], item_empty[kTcItemSlots];
    uint64_t stolen_bar;
    alignas(16) uint4 stolen;                  // answer of the launch unit: the block that will not be launched
    TcItem items[kTcItemSlots];                // nt < 0: no more
    float xm[2][128], xl[2][128];
};
static_assert(sizeof(TcShared) <= kTcBookBytes, "");

template <int D, bool F32, bool TINY, typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
paged_chunk_tc5_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcShape p,
                       const T* __restrict__ q, const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, const uint32_t* __restrict__ tables,
                       const uint32_t* __restrict__ q_starts, const uint32_t* __restrict__ seq_lens, T* __restrict__ out,
                       float* __restrict__ part_o, float2* __restrict__ part_ml, uint32_t* err) {
    using Cfg = TcCfg<D, F32>;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* q_smem = smem;
    unsigned char* ring = smem + Cfg::kQBytes;
    TcShared& sh = *reinterpret_cast<TcShared*>(smem + Cfg::kQBytes + Cfg::kStages * Cfg::kTileBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t q_addr = smem_u32(q_smem), ring_addr = smem_u32(ring);
    constexpr int kNst = Cfg::kStages;
    constexpr int kHalves = D / 64;
    constexpr int kHalfBytes = kTcKeys * 128;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kNst; ++i) {
            mbar_init(smem_u32(&sh.full[0][i]), 1);
            mbar_init(smem_u32(&sh.full[1][i]), 1);
            mbar_init(smem_u32(&sh.empty[i]), 2);      // both slots, or one slot twice
            mbar_init(smem_u32(&sh.raw[i]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&sh.s_full[s]), 1);
            mbar_init(smem_u32(&sh.p_full[s][0]), 4);
            mbar_init(smem_u32(&sh.p_full[s][1]), 4);
            mbar_init(smem_u32(&sh.p_free[s]), 1);
            mbar_init(smem_u32(&sh.o_full[s]), 1);
            mbar_init(smem_u32(&sh.q_full[s]), 4);
            mbar_init(smem_u32(&sh.meet[s]), 4);
        }
        mbar_init(smem_u32(&sh.meet_all), kTcSoftmaxWarps);
        mbar_init(smem_u32(&sh.stolen_bar), 1);
        for (int i = 0; i < 4; ++i) sh.turn[i] = 0;
        for (int i = 0; i < kTcItemSlots; ++i) {
            mbar_init(smem_u32(&sh.item_full[i]), 1);
            mbar_init(smem_u32(&sh.item_empty[i]), kTcSoftmaxWarps + 3);
        }
        fence_barrier_init();
    }
    if (warp == 8 && lane == 0) {
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    // The tensor memory is taken after the wait: a block of the kernel before that has yet to take its own must not find it gone.
    pdl_wait();
    if (warp == 9) {
        tmem_alloc(smem_u32(&sh.tmem), 512);
        tmem_relinquish();
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_launch_dependents();

    const int block = p.sh.block_size;
    // the barrier of the tile at place `at` of the ring, and the parity of its phase
    auto full_bar = [&](uint32_t at) { return &sh.full[(at / kNst) & 1][at % kNst]; };
    auto full_parity = [](uint32_t at) { return (at / (2 * kNst)) & 1; };
    // the k-th item, for every warp but the one that deals them out; null: no more (or the wait ran out)
    auto next_item = [&](uint32_t k) -> TcItem* {
        const uint32_t slot = k % kTcItemSlots;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.item_full[slot]), (k / kTcItemSlots) & 1, err, kErrProducerWait))) return nullptr;
        return sh.items[slot].nt < 0 ? nullptr : &sh.items[slot];
    };
    auto release_item = [&](uint32_t k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.item_empty[k % kTcItemSlots]));
    };

    if (warp >= kTcSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
        // ------------------------------------------------------------ TMA producer: lane i fetches the i-th cache block of a tile
        uint32_t pos = 0, issued = 0, raw_last = 0, raw_phase = 0;      // per stage: its last tile went to `raw`; parity of those
        bool ok = true;
        const int box = min(block, kTcKeys);
        TcWalk<Cfg::kRows, F32> walk(p, q_starts, seq_lens);
        TcItem it;
        uint32_t k_item = 0;
        auto deal = [&]() {
            const uint32_t slot = k_item % kTcItemSlots;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.item_empty[slot]), ((k_item / kTcItemSlots) & 1) ^ 1, err, kErrProducerWait))) return false;
            if (lane == 0) sh.items[slot] = it;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.item_full[slot]));
            ++k_item;
            return true;
        };
        // One block per item in the grid; a block that is through with its own takes over one that has not started, so the items
        // spread evenly whatever their lengths.
        int64_t index = blockIdx.x;
        uint32_t asked = 0, answered = 0;      // requests to the launch unit, and answers taken: at most one is on its way
        while (ok) {
            if (asked > answered) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.stolen_bar), answered & 1, err, kErrProducerWait));
                if (!ok) break;
                ++answered;
                index = stolen_block(smem_u32(&sh.stolen));
                if (index < 0) break;
                fence_proxy_async();
                __syncwarp();
            }
            if (lane == 0) steal_block(smem_u32(&sh.stolen), smem_u32(&sh.stolen_bar));
            ++asked;
            if (!walk.get(index, it, err) || it.nt == 0) continue;
            ok = deal();
            if (!ok) break;
            const TcOrder order(pos, it);
            const uint32_t* table = tables + int64_t(it.seq) * p.sh.max_blocks_per_seq;
            const int end = min(it.max_limit, (it.t0 + it.nt) * kTcKeys);
            const int masked_from = it.min_limit / kTcKeys;
            auto fetch = [&](const CUtensorMap& map, int t, uint32_t at, bool values) {
                const int stage = at % kNst, k0 = (it.t0 + t) * kTcKeys;
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.empty[stage]), ((at / kNst) & 1) ^ 1, err, kErrProducerWait))) return false;
                issued = at + 1;
                const int boxes = (min(kTcKeys, end - k0) + box - 1) / box;
                const bool masked = values && it.t0 + t >= masked_from;
                const uint32_t bar = smem_u32(masked ? &sh.raw[stage] : full_bar(at));
                if (masked) { raw_last |= 1u << stage; raw_phase ^= 1u << stage; }
                else raw_last &= ~(1u << stage);
                if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box * D * 2);
                __syncwarp();
                if (lane < boxes) {
                    const int key = k0 + lane * box;
                    uint32_t blk = table[key / block];
                    if (blk >= uint32_t(p.sh.num_blocks)) {
                        atomicCAS(err, 0u, static_cast<uint32_t>(kErrAttnBlockId));
                        blk = 0;
                    }
                    const int y = int(blk) * block + key % block;
                    const uint32_t dst = ring_addr + stage * Cfg::kTileBytes + lane * box * 128;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) tma_load_2d(dst + h * kHalfBytes, &map, bar, it.kvh * D + h * 64, y);
                }
                return true;
            };
            for (int t = 0; ok && t < order.ahead; ++t) ok = fetch(map_k, t, order.k(t), false);
            for (int t = 0; ok && t < it.nt; ++t) {
                ok = fetch(map_v, t, order.v(t), true);
                if (ok && t + order.ahead < it.nt) ok = fetch(map_k, t + order.ahead, order.k(t + order.ahead), false);
            }
            pos += 2 * it.nt;
        }
        if (ok) {
            it.nt = -1;
            deal();
        }
        // given up: the answer on its way still lands in this block's shared memory
        if (asked > answered) mbar_wait(smem_u32(&sh.stolen_bar), answered & 1, err, kErrProducerWait);
        if (!ok)      // the consumer is gone: let this warp's own copies land before the memory is given back
            for (uint32_t at = issued > kNst ? issued - kNst : 0; at < issued; ++at) {
                const uint32_t stage = at % kNst;
                if ((raw_last >> stage) & 1) mbar_wait(smem_u32(&sh.raw[stage]), ((raw_phase >> stage) & 1) ^ 1, err, kErrProducerWait);
                else mbar_wait(smem_u32(full_bar(at)), full_parity(at), err, kErrProducerWait);
            }
    } else if (warp <= 10) {
        // ------------------------------------------------------------ MMA issue for slot `s` (one elected thread)
        constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((kTcKeys >> 3) << 17) | ((128 >> 4) << 24);
        constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((D >> 3) << 17) | ((128 >> 4) << 24);
        const uint32_t idesc_s = kIdescS | (!F32 && p.q_sign < 0.0f ? 1u << 13 : 0u);      // bit 13: the A operand negated
        const int s = warp - 9;
        const uint32_t d_s = tmem + s * 128, d_o = tmem + 256 + s * 128;
        uint32_t pos = 0, p_phase = 0, k_item = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return bool(__all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, err, kErrMmaWait))); };
        for (TcItem* item; ok && (item = next_item(k_item)) != nullptr; ++k_item) {
            const TcOrder order(pos, *item);
            const int n = item->nt;
            const bool split = TINY || item->split, stack = F32 && (TINY || item->stack);
            release_item(k_item);
            pos += 2 * n;
            // (the other group's part last: it is at most one item behind once this group has stored its part)
            ok = wait(&sh.q_full[s], k_item & 1) && (!split || wait(&sh.q_full[s ^ 1], k_item & 1));
            tc5_fence_after();
            const uint64_t q_desc = umma_desc_k128(q_addr + (F32 || split ? 0 : s) * Cfg::kQTileBytes);
            const int step = split ? 2 : 1;
            // No tile of this item for this slot: its group waits for o_full all the same, since a group that went on to the next item
            // could complete its q_full again before this warp has seen the last one, and the parity wait above would never end.
            if (ok && split && s >= n && elect_one()) mbar_arrive(smem_u32(&sh.o_full[s]));
            __syncwarp();
            // a stage is free when both slots are done with it; a slot that has it for itself says so twice
            auto release = [&](uint32_t stage) {
                tc5_commit(smem_u32(&sh.empty[stage]));
                if (split) tc5_commit(smem_u32(&sh.empty[stage]));
            };
            for (int t = split ? s : 0, nth = 0; ok && t < n; t += step, ++nth) {
                {
                    const uint32_t at = order.k(t), stage = at % kNst;
                    ok = wait(full_bar(at), full_parity(at));
                    if (!ok) break;
                    tc5_fence_after();
                    const uint64_t k_desc = umma_desc_k128(ring_addr + stage * Cfg::kTileBytes);
                    auto multiply = [&](auto terms) {
                        if (elect_one()) {
#pragma unroll
                            for (int left = decltype(terms)::value - 1; left >= 0; --left)      // the small terms first: every step cuts to the sum's precision
#pragma unroll
                                for (int kk = 0; kk < D / 16; ++kk) {
                                    constexpr int kTerms = decltype(terms)::value;
                                    const int term = left;
                                    const uint32_t off = ((kk / 4) * kHalfBytes + (kk % 4) * 32) >> 4;
                                    umma_bf16_ss(d_s, q_desc + off + ((term * Cfg::kQTileBytes) >> 4), k_desc + off, idesc_s, term < kTerms - 1 || kk > 0);
                                }
                            tc5_commit(smem_u32(&sh.s_full[s]));
                            release(stage);
                        }
                        __syncwarp();
                    };
                    multiply(std::integral_constant<int, TINY ? 1 : Cfg::kQTerms>());
                }
                const uint32_t at = order.v(t), stage = at % kNst;
                ok = wait(full_bar(at), full_parity(at));
                const uint64_t v_desc = umma_desc_mn128(ring_addr + stage * Cfg::kTileBytes, kHalfBytes);
                // not the first product of this item, nor the first after O was put aside
                if (F32 && !TINY && nth == (stack ? Cfg::kHoldStack : Cfg::kHold)) nth = 0;
                const uint32_t keep = nth > 0;
                const bool last = t + step >= n;
                auto multiply = [&](auto half, auto terms) {
                    constexpr int kTerms = decltype(terms)::value, H = decltype(half)::value;
                    if (elect_one()) {
#pragma unroll
                        for (int left = kTerms - 1; left >= 0; --left)      // the small terms first, as above
#pragma unroll
                            for (int kk = 0; kk < kTcKeys / 16; ++kk) {
                                const int term = left;
                                constexpr int kFirst = F32 ? 4 : 6;            // products of 16 keys in the first part
                                if ((kk < kFirst) != (H == 0)) continue;
                                const uint32_t cols = kTerms == 3 ? weight_columns<D>(H, term) + (kk - H * kFirst) * 8 : kk * 8;
                                umma_bf16_ts(d_o, d_s + cols, v_desc + ((kk * 2048) >> 4), kIdescO, term < kTerms - 1 || kk > 0 ? 1u : keep);
                            }
                        if (H == 0 && kTerms == 3 && D == 128) tc5_commit(smem_u32(&sh.p_free[s]));
                        if (H == 1) {
                            if (last) tc5_commit(smem_u32(&sh.o_full[s]));
                            release(stage);
                        }
                    }
                    __syncwarp();
                };
                using One = std::integral_constant<int, 1>;
                using Zero = std::integral_constant<int, 0>;
                using All = std::integral_constant<int, Cfg::kPTerms>;
                ok = ok && wait(&sh.p_full[s][0], p_phase & 1);
                if (!ok) break;
                tc5_fence_after();
                if constexpr (TINY) multiply(Zero(), One());
                else if (F32 && stack) multiply(Zero(), One());
                else multiply(Zero(), All());
                ok = wait(&sh.p_full[s][1], p_phase & 1);
                if (!ok) break;
                tc5_fence_after();
                if constexpr (TINY) multiply(One(), One());
                else if (F32 && stack) multiply(One(), One());
                else multiply(One(), All());
                ++p_phase;
            }
        }
    } else {
        // ------------------------------------------------------------ V tiles with masked keys
        uint32_t pos = 0, raw_phase = 0, k_item = 0;
        bool ok = true;
        for (TcItem* item; ok && (item = next_item(k_item)) != nullptr; release_item(k_item++)) {
            const TcItem& it = *item;
            const TcOrder order(pos, it);
            pos += 2 * it.nt;
            const int masked_from = it.min_limit / kTcKeys;
            for (int t = max(0, masked_from - it.t0); ok && t < it.nt; ++t) {
                const uint32_t at = order.v(t), stage = at % kNst;
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.raw[stage]), (raw_phase >> stage) & 1, err, kErrAttnLoadWait));
                if (!ok) break;
                raw_phase ^= 1u << stage;
                const int k0 = (it.t0 + t) * kTcKeys;
                unsigned char* tile = ring + stage * Cfg::kTileBytes;
                bool found = false;
                // rows some query must not see, then rows nobody sees; 8 pieces of 16 bytes are a row of a half
                const int r0 = max(0, it.min_limit - k0), r1 = min(kTcKeys, it.max_limit - k0);
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    uint4* pieces = reinterpret_cast<uint4*>(tile + h * kHalfBytes);
                    for (int c0 = r0 * 8; c0 < r1 * 8; c0 += 256) {
                        uint4 v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = c0 + k * 32 + lane < r1 * 8 ? pieces[c0 + k * 32 + lane] : make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
                            bool bad = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((w[e] & 0x7F80u) == 0x7F80u) { w[e] &= 0xFFFF0000u; bad = true; }
                                if ((w[e] & 0x7F800000u) == 0x7F800000u) { w[e] &= 0x0000FFFFu; bad = true; }
                            }
                            if (bad) { pieces[c0 + k * 32 + lane] = v[k]; found = true; }
                        }
                    }
#pragma unroll 8
                    for (int c = r1 * 8 + lane; c < kTcKeys * 8; c += 32) pieces[c] = make_uint4(0, 0, 0, 0);
                }
                if (found) item->nonfinite = 1;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(full_bar(at)));
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ------------------------------------------------------------ softmax: group `wg` of four warps, thread = row
        const int wg = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lane_base = uint32_t(warp & 3) << 21;               // 32 lanes a warp, lane field in the upper half of the address
        const uint32_t t_s = tmem + wg * 128 + lane_base, t_o = tmem + 256 + wg * 128 + lane_base;
        const float c = p.scale_log2;
        uint32_t s_phase = 0, f_phase = 0, o_phase = 0, k_item = 0, all_phase = 0, wg_phase = 0;      // f_phase: tiles whose first half is waited for (p_free)
        bool ok = true, was_split = true;
        // (mbarriers instead of named barriers: their waits end when somebody has given up)
        auto meet_all = [&]() {
            tc5_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.meet_all));
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.meet_all), all_phase++ & 1, err, kErrEpilogueWait)) && ok;
            tc5_fence_after();
        };
        auto meet_group = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.meet[wg]));
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.meet[wg]), wg_phase++ & 1, err, kErrEpilogueWait)) && ok;
        };
        // Warps w and w + 4 share an exponential unit.  Left alone they fall into step - both exponentiate while the tensor cores
        // wait, then both wait - so one lets the other finish first.  A courtesy with a limit: nothing depends on it.
        bool my_turn = false;
        auto take_turn = [&]() {
            if (lane == 0) {
                for (int i = 0; i < 48 && !my_turn; ++i) my_turn = atomicExch(&sh.turn[warp & 3], 1u) == 0u;
            }
            __syncwarp();
        };
        auto end_turn = [&]() {
            if (lane == 0 && my_turn) atomicExch(&sh.turn[warp & 3], 0u);
            my_turn = false;
        };
        for (TcItem* item; ok && (item = next_item(k_item)) != nullptr; release_item(k_item++)) {
            const TcItem& it = *item;
            const bool stack = F32 && !TINY && it.stack, split = TINY || it.split;
            constexpr int kTiny = Cfg::kTinyRows;
            const int r = TINY ? lane % kTiny : (stack ? row & 31 : (split ? 0 : wg * 128) + row);      // row of the item
            const bool live = r < it.rows && (!TINY || lane < Cfg::kQTerms * kTiny);
            // a warp without rows only keeps the barriers going: its accumulator rows hold garbage that nobody reads
            const bool busy = __any_sync(0xffffffffu, live) && !(stack && (warp & 3) == 3);
            const int list = it.row0 + r, token = list / p.group, head = it.kvh * p.group + list % p.group;
            const int limit = live ? it.len - it.n + token + 1 : 0;
            const int64_t out_row = (int64_t(it.start) + token) * p.sh.num_q_heads + head;

            // The query tiles are free: a group that has its slot to itself waits for its own warps only, and so works through its
            // items independently of the other group.
            if (!split) meet_group();
            else if (!was_split) meet_all();
            was_split = split;
            if (!ok) break;

            // Queries into shared memory, 128-byte swizzled.  A warp reads whole rows (a lane 8 elements of one), several before it
            // uses the first; a tile that both slots use is shared out over all eight warps.
            {
                constexpr int kPieces = D / 8, kAtOnce = 32 / kPieces, kBatch = 2;
                const int per = stack || TINY ? 4 : (split ? 16 : 32), base = (split ? warp : warp & 3) * per;
                const int first = (split ? 0 : wg * 128) + base, count = min(per, it.rows - first);      // rows of this warp (<= 0: none)
                // place of the row base + lane; rows that the item does not have read its first row and are set to zero
                const int at = it.row0 + (lane < count ? first + lane : 0), tok = at / p.group;
                const int64_t from = (int64_t(it.start) + tok) * p.sh.row_stride + int64_t(it.kvh * p.group + at - tok * p.group) * D;
                const int piece = lane % kPieces;
                unsigned char* dst = q_smem + (split ? 0 : wg) * Cfg::kQTileBytes + (piece / 8) * kHalfBytes;
                if constexpr (!F32) {      // straight into shared memory, all of it in flight at once
#pragma unroll 1
                    for (int j = lane / kPieces; j < per; j += kAtOnce) {
                        const int64_t f = __shfl_sync(0xffffffffu, static_cast<long long>(from), j & 31);
                        const int to = base + j;
#pragma unroll
                        for (int quarter = 0; quarter < (TINY ? 4 : 1); ++quarter) {
                            const int tr = quarter * 32 + to;
                            copy_async_16(smem_u32(dst + tr * 128 + (((piece % 8) ^ (tr & 7)) << 4)), q + f + piece * 8, j < count);
                        }
                    }
                    copy_async_wait();
                } else {
#pragma unroll 1
                for (int j0 = lane / kPieces; j0 < per; j0 += kBatch * kAtOnce) {
                    using Raw = Pack<T, 8>;
                    Raw raw[kBatch];
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                        const int64_t f = __shfl_sync(0xffffffffu, static_cast<long long>(from), (j0 + b * kAtOnce) & 31);
                        const uint4* src = reinterpret_cast<const uint4*>(q + f + piece * 8);
#pragma unroll
                        for (int k = 0; k < int(sizeof(Raw) / 16); ++k) reinterpret_cast<uint4*>(&raw[b])[k] = __ldg(src + k);
                    }
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                        const int j = j0 + b * kAtOnce, to = base + j, sw = ((piece % 8) ^ (to & 7)) << 4;
                        const float sign = j < count ? p.q_sign : 0.0f;
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[k] = j < count ? as_f32(raw[b].v[k]) * sign : 0.0f;
#pragma unroll
                        for (int term = 0; term < Cfg::kQTerms; ++term) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                w[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
                                x[2 * k] -= bf16_lo(w[k]);
                                x[2 * k + 1] -= bf16_hi(w[k]);
                            }
                            unsigned char* tile = dst + term * Cfg::kQTileBytes;
                            if constexpr (TINY) {
                                if (j < per && to < kTiny) {
#pragma unroll
                                    for (int quarter = 0; quarter < 4; ++quarter) {
                                        const int tr = quarter * 32 + term * kTiny + to;
                                        *reinterpret_cast<uint4*>(dst + tr * 128 + (((piece % 8) ^ (tr & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                                    }
                                }
                            }
                            if (!TINY && j < per) *reinterpret_cast<uint4*>(tile + to * 128 + sw) = make_uint4(w[0], w[1], w[2], w[3]);
                            if (!TINY && stack && j < per) {
                                *reinterpret_cast<uint4*>(tile + (32 + to) * 128 + sw) = make_uint4(w[0], w[1], w[2], w[3]);
                                *reinterpret_cast<uint4*>(tile + (64 + to) * 128 + sw) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                }
                }
                fence_proxy_async();
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[wg]));
            }

            float m = -INFINITY, l = 0.0f;
            // f32 activations: the MMAs cut their sums towards zero, up to the last bit at each of a tile's additions (24 for three terms of 128
            // keys), so an accumulator loses about 1.4e-8 of itself each time.  After 48 additions - two tiles, or six of a stacked item -
            // its row is therefore put aside, in local memory, and added up by f32 additions that round.  512 tokens over 8000, in
            // 1e-6 off and us: 13.9 and 356 without; 1.9 and 392 every four tiles, 1.5 and 406 every three, 1.1 and 434 every two, 0.7
            // and 567 every tile; plain f32 operations 0.9.
            // (The warps of few rows add two products of their own keys a tile; their key ranges are short enough, see plan_chunk.)
            constexpr bool kHolds = F32 && !TINY;
            const int hold = stack ? Cfg::kHoldStack : Cfg::kHold;
            [[maybe_unused]] float held[kHolds ? D : 1], held_m = 0.0f;
            [[maybe_unused]] int since = 0;
            [[maybe_unused]] bool some = false;
            // O and what was put aside (if anything was), 16 columns at a time, the next ones already on their way
            [[maybe_unused]] auto add_held = [&](auto put) {
                const float f = held_m == m ? 1.0f : ex2((held_m - m) * c);
                float next[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) next[k] = some ? held[k] : 0.0f;
#pragma unroll 1
                for (int g = 0; g < D; g += 16) {
                    float sum[16];
                    uint32_t o[16];
                    tmem_ld_32x16(t_o + g, o);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        sum[k] = next[k];
                        if (some && g + 16 < D) next[k] = held[g + 16 + k];
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; ++k) sum[k] = some ? fmaf(sum[k], f, __uint_as_float(o[k])) : __uint_as_float(o[k]);
                    put(g, sum);
                }
            };
            const int masked_from = it.min_limit / kTcKeys - it.t0, step = split ? 2 : 1, nt = it.nt, k0 = it.t0 * kTcKeys;
            int done = 0;
            for (int t = split ? wg : 0; t < nt; t += step, ++done) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.s_full[wg]), s_phase & 1, err, kErrEpilogueWait));
                if (!ok) break;
                if (!busy) {
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_u32(&sh.p_full[wg][0]));
                        mbar_arrive(smem_u32(&sh.p_full[wg][1]));
                    }
                    ++s_phase;
                    f_phase += !stack;
                    continue;
                }
                tc5_fence_after();
                if constexpr (kHolds) {      // (the products before this one's scores are complete)
                    if (since++ == hold) {
                        add_held([&](int col, const float (&sum)[16]) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) held[col + k] = sum[k];
                        });
                        some = true;
                        since = 1;
                        held_m = m;
                    }
                }
                const bool masked = t >= masked_from;                          // the same for all lanes, as the collective loads and stores need
                const int visible = limit - k0 - t * kTcKeys;
                // Running maximum; true when O was rescaled.  m may stay behind by 2^8 in the weight.
                auto raise = [&](float top) {
                    if (done == 0) {
                        m = top;
                    } else if (__any_sync(0xffffffffu, !((top - m) * c <= 8.0f))) {
                        const float m_new = max_nan(m, top);
                        const float f = m_new == m ? 1.0f : ex2((m - m_new) * c);
                        m = m_new;
                        l *= f;
#pragma unroll 1
                        for (int g = 0; g < D / 16; ++g) {
                            uint32_t o[16];
                            tmem_ld_32x16(t_o + g * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st_32x16(t_o + g * 16, o);
                        }
                    }
                };
                F2 sum[2] = {F2(0.0f, 0.0f), F2(0.0f, 0.0f)};
                if constexpr (TINY) {
                    const int key0 = (warp & 3) * 32;
                    uint32_t raw[32];
                    tmem_ld_32x32(t_s + key0, raw);
                    tmem_ld_wait();
                    if constexpr (F32) {      // the three partial scores, added in the same order by all three lanes
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const float v = __uint_as_float(raw[k]);
                            const float a = __shfl_sync(0xffffffffu, v, r), b = __shfl_sync(0xffffffffu, v, r + 10), d = __shfl_sync(0xffffffffu, v, r + 20);
                            raw[k] = __float_as_uint((d + b) + a);
                        }
                    }
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (key0 + k >= visible) raw[k] = 0xFF800000u;
                    }
                    float mx[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        mx[g] = max_nan(__uint_as_float(raw[g]), __uint_as_float(raw[g + 4]));
#pragma unroll
                        for (int k = 8; k < 32; k += 8) mx[g] = max_nan(mx[g], __uint_as_float(raw[k + g]), __uint_as_float(raw[k + g + 4]));
                    }
                    float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
                    if constexpr (F32) {
                        // Infinities of K or q: the small terms of a query make NaN of them (0 inf, inf - inf), the first term alone does not
                        if (__any_sync(0xffffffffu, live && top != top)) {
                            tmem_ld_32x32(t_s + key0, raw);
                            tmem_ld_wait();
                            top = -INFINITY;
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                const float v = __uint_as_float(raw[k]);
                                const float a = __shfl_sync(0xffffffffu, v, r), b = __shfl_sync(0xffffffffu, v, r + 10), d = __shfl_sync(0xffffffffu, v, r + 20);
                                float x = (d + b) + a;
                                x = masked && key0 + k >= visible ? -INFINITY : (x != x ? a : x);
                                top = max_nan(top, x);
                                raw[k] = __float_as_uint(x);
                            }
                        }
                    }
                    raise(top);
                    const float mc = m == -INFINITY ? 0.0f : (m == INFINITY ? __int_as_float(0x7FC00000) : m * c);
                    const F2 c2(c, c), mc2(-mc, -mc);
                    const int term = F32 ? lane / kTiny : 0;
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float a, b;
                        fma2(F2(__uint_as_float(raw[k]), __uint_as_float(raw[k + 1])), c2, mc2).get(a, b);
                        a = ex2(a);
                        b = ex2(b);
                        sum[(k / 2) & 1] = add2(sum[(k / 2) & 1], F2(a, b));
                        if constexpr (F32) {
                            uint32_t w0 = cut_bf16(a, b);
                            cut_rest(a, b).get(a, b);
                            const uint32_t w1 = cut_bf16(a, b);
                            cut_rest(a, b).get(a, b);
                            w[k / 2] = term == 0 ? w0 : (term == 1 ? w1 : cut_bf16(a, b));
                        } else {
                            w[k / 2] = pack_bf16(a, b);
                        }
                    }
                    tmem_st_32x16(t_s + (warp & 3) * 16, w);
#pragma unroll
                    for (int k = 0; k < 16; ++k) w[k] = 0;
#pragma unroll
                    for (int g = 1; g < 4; ++g) tmem_st_32x16(t_s + ((warp + g) & 3) * 16, w);
                    tmem_st_wait();
                    tc5_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_u32(&sh.p_full[wg][0]));
                        mbar_arrive(smem_u32(&sh.p_full[wg][1]));
                    }
                } else if constexpr (!F32) {
                    float s[128];      // the whole row stays in registers
                    {
                        uint32_t raw[4][32];
                        tmem_ld_32x32(t_s, raw[0]);
                        tmem_ld_32x32(t_s + 32, raw[1]);
                        tmem_ld_32x32(t_s + 64, raw[2]);
                        tmem_ld_32x32(t_s + 96, raw[3]);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 128; ++k) s[k] = __uint_as_float(raw[k / 32][k % 32]);
                    }
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 128; ++k)
                            if (k >= visible) s[k] = -INFINITY;
                    }
                    float mx[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        mx[g] = max_nan(s[g], s[g + 4]);
#pragma unroll
                        for (int k = 8; k < 128; k += 8) mx[g] = max_nan(mx[g], s[k + g], s[k + 4 + g]);
                    }
                    raise(max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])));
                    const float mc = m == -INFINITY ? 0.0f : (m == INFINITY ? __int_as_float(0x7FC00000) : m * c);      // a score of +inf: NaN, as inf - inf is
                    const F2 c2(c, c), mc2(-mc, -mc);
                    take_turn();
#pragma unroll
                    for (int g = 0; g < 4; ++g) {      // 32 keys, 16 columns
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const int at = g * 32 + k;
                            float a, b;
                            fma2(F2(s[at], s[at + 1]), c2, mc2).get(a, b);
                            a = ex2(a);
                            b = ex2(b);
                            sum[(k / 2) & 1] = add2(sum[(k / 2) & 1], F2(a, b));
                            w[k / 2] = pack_bf16(a, b);
                        }
                        tmem_st_32x16(t_s + g * 16, w);
                        if (g == 3) end_turn();
                        if (g >= 2) {                  // 96 keys are handed over, then the other 32
                            tmem_st_wait();
                            tc5_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[wg][g - 2]));
                        }
                    }
                } else {
                    // The scores are read twice, 32 at a time: a row of them and its three terms do not fit the registers together.
                    float top = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        uint32_t raw[2][32];
                        tmem_ld_32x32(t_s + h * 64, raw[0]);
                        tmem_ld_32x32(t_s + h * 64 + 32, raw[1]);
                        tmem_ld_wait();
                        if (masked) {
#pragma unroll
                            for (int k = 0; k < 64; ++k)
                                if (h * 64 + k >= visible) raw[k / 32][k % 32] = 0xFF800000u;
                        }
                        if (masked) {
                            tmem_st_32x32(t_s + h * 64, raw[0]);
                            tmem_st_32x32(t_s + h * 64 + 32, raw[1]);
                        }
                        float mx[4];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            mx[g] = max_nan(__uint_as_float(raw[0][g]), __uint_as_float(raw[0][g + 4]));
#pragma unroll
                            for (int k = 8; k < 64; k += 8)
                                mx[g] = max_nan(mx[g], __uint_as_float(raw[(k + g) / 32][(k + g) % 32]), __uint_as_float(raw[(k + g + 4) / 32][(k + g + 4) % 32]));
                        }
                        top = max_nan(top, max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])));
                    }
                    tmem_st_wait();
                    // The same for the other items, whose terms are added up by the MMA: such scores are computed again
                    if (__any_sync(0xffffffffu, live && top != top)) {
                        top = -INFINITY;
#pragma unroll 1
                        for (int k = 0; k < kTcKeys; ++k) {
                            float x = __uint_as_float(tmem_ld_32x1(t_s + k));
                            tmem_ld_wait();
                            if (live && x != x) {
                                const int key = k0 + t * kTcKeys + k;
                                const uint32_t blk = min(tables[int64_t(it.seq) * p.sh.max_blocks_per_seq + key / block], uint32_t(p.sh.num_blocks - 1));
                                const uint16_t* kr = k_pool + (int64_t(blk) * block + key % block) * (int64_t(p.sh.num_kv_heads) * D) + it.kvh * D;
                                const T* qr = q + (int64_t(it.start) + token) * p.sh.row_stride + int64_t(head) * D;
                                x = 0.0f;
#pragma unroll 1
                                for (int d = 0; d < D; ++d) x = fmaf(as_f32(qr[d]) * p.q_sign, bf16_bits_to_f32(kr[d]), x);
                            }
                            tmem_st_32x1(t_s + k, __float_as_uint(x));
                            top = max_nan(top, x);
                        }
                        tmem_st_wait();
                    }
                    raise(top);
                    const float mc = m == -INFINITY ? 0.0f : (m == INFINITY ? __int_as_float(0x7FC00000) : m * c);      // a score of +inf: NaN, as inf - inf is
                    const F2 c2(c, c), mc2(-mc, -mc);
                    // a half's terms are stored when its own scores, and those that they overwrite, are in registers
                    uint32_t sc[4][32];
                    tmem_ld_32x32(t_s, sc[0]);
                    tmem_ld_32x32(t_s + 32, sc[1]);
                    tmem_ld_32x32(t_s + 64, sc[2]);
                    tmem_ld_wait();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h == 1) {
                            tmem_ld_32x32(t_s + 96, sc[3]);
                            tmem_ld_wait();
                        }
#pragma unroll
                        for (int g = 0; g < 2; ++g) {          // 32 keys, 16 columns a term
                            const uint32_t (&now)[32] = sc[h * 2 + g];
                            uint32_t w[3][16];
#pragma unroll
                            for (int k = 0; k < 32; k += 2) {
                                float a, b;
                                fma2(F2(__uint_as_float(now[k]), __uint_as_float(now[k + 1])), c2, mc2).get(a, b);
                                a = ex2(a);
                                b = ex2(b);
                                sum[(k / 2) & 1] = add2(sum[(k / 2) & 1], F2(a, b));
                                w[0][k / 2] = cut_bf16(a, b);
                                cut_rest(a, b).get(a, b);
                                w[1][k / 2] = cut_bf16(a, b);
                                cut_rest(a, b).get(a, b);
                                w[2][k / 2] = cut_bf16(a, b);
                            }
                            if (stack) {
                                if ((warp & 3) == 0) tmem_st_32x16(t_s + h * 32 + g * 16, w[0]);
                                else if ((warp & 3) == 1) tmem_st_32x16(t_s + h * 32 + g * 16, w[1]);
                                else tmem_st_32x16(t_s + h * 32 + g * 16, w[2]);
                            } else {
                                tmem_st_32x16(t_s + weight_columns<D>(h, 0) + g * 16, w[0]);
                                if (D == 128 && h == 1 && g == 0) {      // the columns of the first half's last two terms
                                    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.p_free[wg]), f_phase & 1, err, kErrEpilogueWait)) && ok;
                                    tc5_fence_after();
                                }
                                tmem_st_32x16(t_s + weight_columns<D>(h, 1) + g * 16, w[1]);
                                tmem_st_32x16(t_s + weight_columns<D>(h, 2) + g * 16, w[2]);
                            }
                        }
                        tmem_st_wait();
                        tc5_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[wg][h]));
                    }
                }
                ++s_phase;
                f_phase += !stack;
                float a, b;
                add2(sum[0], sum[1]).get(a, b);
                l += a + b;
                if (!ok) break;
            }
            if (ok) {      // done == 0 too: its slot has then seen the queries' barriers, see there
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.o_full[wg]), o_phase & 1, err, kErrEpilogueWait));
                ++o_phase;
                tc5_fence_after();
            }
            if (!ok) break;
            if constexpr (kHolds) {
                if (some) {      // what was put aside comes back
                    add_held([&](int col, const float (&sum)[16]) {
                        uint32_t o[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(sum[k]);
                        tmem_st_32x16(t_o + col, o);
                    });
                    tmem_st_wait();
                }
            }

            // ---- results.  Rows go through shared memory (the query tiles are done with), so that a warp writes whole rows:
            // row r of a staging area of W-element rows keeps its 16-byte piece j at piece j ^ (r & 7).
            const bool direct = it.nchunks == 1;
            bool patch = false;
            // A row's reach (visible keys) as the warps hand it round: negative where the sum of its weights is no positive number, so that
            // its results mean what they are.
            int reach = limit;
            auto weigh = [&](float sum) { reach = sum > 0.0f && sum < INFINITY ? limit : -limit; };
            // Finishes N columns of the row with this place and reach.  Infinities and NaN of V that the row sees: the MMAs did not get
            // those of cleaned tiles, and made NaN of the others where they met weights of zero (the terms of a weight, the keys of the
            // other warps, a sum scaled down to nothing).  The definition has the values themselves, so such a column is put together again.
            auto finish = [&](int64_t to_row, int seen, int col, auto& o) {
                constexpr int N = sizeof(o) / sizeof(float);
                bool look = patch;
#pragma unroll
                for (int k = 0; k < N; ++k) look |= o[k] != o[k];
                if (look && seen > 0) {
                    float extra[N];
#pragma unroll
                    for (int k = 0; k < N; ++k) extra[k] = 0.0f;
                    const int to = min(seen, k0 + nt * kTcKeys);
#pragma unroll 1
                    for (int j = k0; j < to; ++j) {
                        const uint32_t blk = tables[int64_t(it.seq) * p.sh.max_blocks_per_seq + j / block];
                        if (blk >= uint32_t(p.sh.num_blocks)) continue;
                        const uint16_t* v = v_pool + (int64_t(blk) * block + j % block) * (int64_t(p.sh.num_kv_heads) * D) + it.kvh * D + col;
#pragma unroll
                        for (int k = 0; k < N; ++k)
                            if ((v[k] & 0x7F80u) == 0x7F80u) extra[k] += bf16_bits_to_f32(v[k]);
                    }
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        if (extra[k] != 0.0f) o[k] = (o[k] != o[k] ? 0.0f : o[k]) + extra[k];
                }
                if (direct) store_f32<T, N>(out + to_row * D + col, o);
                else store_f32<float, N>(part_o + (to_row * p.max_chunks + it.chunk) * D + col, o);
            };
            auto row_of = [&](int j) { return static_cast<int64_t>(__shfl_sync(0xffffffffu, static_cast<long long>(out_row), j)); };
            auto reach_of = [&](int j) { return __shfl_sync(0xffffffffu, reach, j); };
            // The rows [j, j + 32 / kLanes, ...) of a warp's 32, kLanes lanes of N columns to a row: all in flight together.  `get`
            // reads the staged columns of a row.
            auto write_rows = [&](auto lanes, auto columns, int col0, auto get) {
                constexpr int kLanes = decltype(lanes)::value, N = decltype(columns)::value, kAtOnce = 32 / kLanes, kSteps = 32 / kAtOnce;
                constexpr int kBatch = kSteps < 2 ? kSteps : 2;
                const int col = lane % kLanes * N;
#pragma unroll 1
                for (int j0 = 0; j0 < 32; j0 += kBatch * kAtOnce) {
                    float o[kBatch][N];
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) get(j0 + b * kAtOnce + lane / kLanes, col, o[b]);
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                        const int j = j0 + b * kAtOnce + lane / kLanes, seen = reach_of(j);
                        const int64_t to_row = row_of(j);
                        if (seen != 0) finish(to_row, seen, col0 + col, o[b]);
                    }
                }
            };
            auto staged = [&](unsigned char* area, int width, int rr, int col) -> float4* {
                return reinterpret_cast<float4*>(area + (size_t(rr) * width + (((col >> 2) ^ (rr & 7)) << 2)) * 4);
            };
            if (!TINY && !split) {
                if constexpr (!F32 && !TINY) {
                    patch = *reinterpret_cast<volatile uint32_t*>(&item->nonfinite) != 0;      // set before the products that o_full stands for
                    const float inv = direct ? 1.0f / l : 1.0f;
                    weigh(l);
                    unsigned char* area = q_smem + wg * Cfg::kQTileBytes + (warp & 3) * (Cfg::kQTileBytes / 4);
                    bool plain = direct && !patch;
                    if (plain && busy) {      // 32 finished bf16 rows fit this warp's part of its group's query tile
                        uint32_t nan = 0;
#pragma unroll 1
                        for (int g = 0; g < D / 32; ++g) {
                            uint32_t raw[32];
                            tmem_ld_32x32(t_o + g * 32, raw);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 32; k += 8) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    w[e] = pack_bf16(__uint_as_float(raw[k + 2 * e]) * inv, __uint_as_float(raw[k + 2 * e + 1]) * inv);
                                    nan = max_nan_bf16(nan, w[e]);
                                }
                                *reinterpret_cast<uint4*>(area + lane * (D * 2) + (((g * 4 + k / 8) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        __syncwarp();
                        // a NaN that the weights did not make (the largest of the bf16 that came by): the rows go the other way
                        plain = !__any_sync(0xffffffffu, reach > 0 && ((nan & 0xFFFFu) == 0x7FFFu || nan >> 16 == 0x7FFFu));
                        constexpr int kPieces = D / 8, kAtOnce = 32 / kPieces;
                        const int piece = lane % kPieces;
#pragma unroll 4
                        for (int j = lane / kPieces; plain && j < 32; j += kAtOnce) {
                            const int64_t to_row = row_of(j);
                            const bool there = reach_of(j) != 0;
                            const uint4 v = *reinterpret_cast<const uint4*>(area + j * (D * 2) + ((piece ^ (j & 7)) << 4));
                            if (there) *reinterpret_cast<uint4*>(out + to_row * D + piece * 8) = v;
                        }
                    }
                    __syncwarp();
                    // key ranges and patched rows: 32 rows of 64 f32 columns at a time (D = 64: of 32 columns)
                    constexpr int kCols = D / 2;
#pragma unroll 1
                    for (int part = plain ? 2 : 0; part < 2; ++part) {
                        if (busy) {
#pragma unroll 1
                            for (int g = 0; g < kCols / 32; ++g) {
                                uint32_t raw[32];
                                tmem_ld_32x32(t_o + part * kCols + g * 32, raw);
                                tmem_ld_wait();
#pragma unroll
                                for (int k = 0; k < 32; k += 4)
                                    *staged(area, kCols, lane, g * 32 + k) =
                                        make_float4(__uint_as_float(raw[k]) * inv, __uint_as_float(raw[k + 1]) * inv,
                                                    __uint_as_float(raw[k + 2]) * inv, __uint_as_float(raw[k + 3]) * inv);
                            }
                        }
                        __syncwarp();
                        if (busy)
                            write_rows(std::integral_constant<int, kCols / 8>(), std::integral_constant<int, 8>(), part * kCols, [&](int j, int col, float (&o)[8]) {
                            const float4 x = *staged(area, kCols, j, col), y = *staged(area, kCols, j, col + 4);
                            o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w; o[4] = y.x; o[5] = y.y; o[6] = y.z; o[7] = y.w;
                        });
                        __syncwarp();
                    }
                    if (!direct && live) part_ml[out_row * p.max_chunks + it.chunk] = make_float2(m * c, l);
                }
                tc5_fence_before();
            } else {
                const int lane_row = stack ? lane : row;
                sh.xm[wg][row] = m;
                sh.xl[wg][row] = l;
                meet_all();      // every product that reads the query tile is complete: it may be overwritten
                if (!ok) break;
                patch = *reinterpret_cast<volatile uint32_t*>(&item->nonfinite) != 0;
                if constexpr (TINY) {
                    // Row rr: the sum over slots, warps and terms.  One slot's accumulator rows at a time fit the query tiles.
                    constexpr int kMost = (kTiny + 7) / 8;
                    float o[kMost][4], top[kMost], total[kMost];
                    const int col = lane * 4;
#pragma unroll
                    for (int j = 0; j < kMost; ++j) {
                        const int rr = min(warp + j * 8, kTiny - 1);
                        top[j] = -INFINITY;
                        total[j] = 0.0f;
#pragma unroll
                        for (int x = 0; x < 8; ++x) top[j] = max_nan(top[j], sh.xm[x >> 2][(x & 3) * 32 + rr]);
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const float mx = sh.xm[x >> 2][(x & 3) * 32 + rr];
                            if (mx != -INFINITY) total[j] = fmaf(sh.xl[x >> 2][(x & 3) * 32 + rr], ex2((mx - top[j]) * c), total[j]);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[j][k] = 0.0f;
                    }
#pragma unroll 1
                    for (int from = 0; from < 2; ++from) {
                        if (wg == from && done > 0) {
#pragma unroll
                            for (int g = 0; g < D / 32; ++g) {
                                uint32_t raw[32];
                                tmem_ld_32x32(t_o + g * 32, raw);
                                tmem_ld_wait();
#pragma unroll
                                for (int k = 0; k < 32; k += 4)
                                    *staged(q_smem, D, row, g * 32 + k) = make_float4(__uint_as_float(raw[k]), __uint_as_float(raw[k + 1]),
                                                                                      __uint_as_float(raw[k + 2]), __uint_as_float(raw[k + 3]));
                            }
                        }
                        meet_all();
#pragma unroll
                        for (int j = 0; j < kMost; ++j) {
                            const int rr = warp + j * 8;
                            if (rr >= it.rows || col >= D) continue;
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const float mx = sh.xm[from][x * 32 + rr];
                                if (mx == -INFINITY) continue;      // no key there
                                const float f = ex2((mx - top[j]) * c);
                                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int term = Cfg::kQTerms - 1; term >= 0; --term) {
                                    const float4 y = *staged(q_smem, D, x * 32 + term * kTiny + rr, col);
                                    v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
                                }
#pragma unroll
                                for (int k = 0; k < 4; ++k) o[j][k] = fmaf(v[k], f, o[j][k]);
                            }
                        }
                        meet_all();      // read: the other slot's rows, or the next item's queries, may come
                        if (!ok) break;
                    }
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < kMost; ++j) {
                        const int rr = warp + j * 8, seen = abs(reach_of(min(rr, kTiny - 1)));
                        const int64_t to_row = row_of(min(rr, kTiny - 1));
                        if (rr >= it.rows) continue;
                        if (lane == 0 && !direct) part_ml[to_row * p.max_chunks + it.chunk] = make_float2(top[j] * c, total[j]);
                        const float inv = direct ? 1.0f / total[j] : 1.0f;
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[j][k] *= inv;
                        if (col < D) finish(to_row, total[j] > 0.0f && total[j] < INFINITY ? seen : -seen, col, o[j]);
                    }
                } else {
                const float m0 = sh.xm[0][lane_row], m1 = sh.xm[1][lane_row], mt = fmaxf(m0, m1);
                const float f0 = m0 == -INFINITY ? 0.0f : ex2((m0 - mt) * c), f1 = m1 == -INFINITY ? 0.0f : ex2((m1 - mt) * c);
                const float lt = fmaf(sh.xl[0][lane_row], f0, sh.xl[1][lane_row] * f1);
                const float inv = direct ? 1.0f / lt : 1.0f;
                weigh(lt);
                const float mine = (wg == 0 ? f0 : f1) * inv;
                if (!direct && live && warp == (stack ? 0 : warp & 3)) part_ml[out_row * p.max_chunks + it.chunk] = make_float2(mt * c, lt);
                if (stack) {
                    if (busy) {
#pragma unroll 1
                        for (int g = 0; g < D / 32; ++g) {
                            uint32_t raw[32];
                            if (done > 0) {
                                tmem_ld_32x32(t_o + g * 32, raw);
                                tmem_ld_wait();
                            }
#pragma unroll
                            for (int k = 0; k < 32; k += 4)
                                *staged(q_smem, D, wg * 96 + row, g * 32 + k) =
                                    done > 0 ? make_float4(__uint_as_float(raw[k]) * mine, __uint_as_float(raw[k + 1]) * mine,
                                                           __uint_as_float(raw[k + 2]) * mine, __uint_as_float(raw[k + 3]) * mine)
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                    }
                    meet_all();
                    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;
#pragma unroll
                    for (int j = 0; j < 4; j += kAtOnce) {
                        const int rr = warp * 4 + j + lane / kLanes, col = lane % kLanes * 4, seen = reach_of(rr);
                        const int64_t to_row = row_of(rr);
                        if (seen == 0) continue;
                        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int x = 5; x >= 0; --x) {      // the small terms first
                            const float4 v = *staged(q_smem, D, (x & 1) * 96 + (x >> 1) * 32 + rr, col);
                            o[0] += v.x; o[1] += v.y; o[2] += v.z; o[3] += v.w;
                        }
                        finish(to_row, seen, col, o);
                    }
                } else {
                    // group g finishes the columns [g D/2, (g + 1) D/2): the other group's half through shared memory, scaled
                    constexpr int kCols = D / 2;
                    const int other = wg ^ 1;
                    if (busy) {
#pragma unroll 1
                        for (int g = 0; g < kCols / 32; ++g) {
                            uint32_t raw[32];
                            if (done > 0) {
                                tmem_ld_32x32(t_o + other * kCols + g * 32, raw);
                                tmem_ld_wait();
                            }
#pragma unroll
                            for (int k = 0; k < 32; k += 4)
                                *staged(q_smem + other * 128 * kCols * 4, kCols, row, g * 32 + k) =
                                    done > 0 ? make_float4(__uint_as_float(raw[k]) * mine, __uint_as_float(raw[k + 1]) * mine,
                                                           __uint_as_float(raw[k + 2]) * mine, __uint_as_float(raw[k + 3]) * mine)
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                    }
                    meet_all();
                    unsigned char* area = q_smem + wg * 128 * kCols * 4;
                    if (busy && done > 0) {
#pragma unroll 1
                        for (int g = 0; g < kCols / 32; ++g) {
                            uint32_t raw[32];
                            tmem_ld_32x32(t_o + wg * kCols + g * 32, raw);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                float4* at = staged(area, kCols, row, g * 32 + k);
                                const float4 x = *at;
                                *at = make_float4(fmaf(__uint_as_float(raw[k]), mine, x.x), fmaf(__uint_as_float(raw[k + 1]), mine, x.y),
                                                  fmaf(__uint_as_float(raw[k + 2]), mine, x.z), fmaf(__uint_as_float(raw[k + 3]), mine, x.w));
                            }
                        }
                    }
                    __syncwarp();
                    constexpr int N = F32 ? 4 : 8;
                    if (busy)
                        write_rows(std::integral_constant<int, kCols / N>(), std::integral_constant<int, N>(), wg * kCols, [&](int j, int col, float (&o)[N]) {
#pragma unroll
                            for (int k = 0; k < N; k += 4) {
                                const float4 x = *staged(area, kCols, (warp & 3) * 32 + j, col + k);
                                o[k] = x.x; o[k + 1] = x.y; o[k + 2] = x.z; o[k + 3] = x.w;
                            }
                        });
                }
                meet_all();      // the exchanged halves have been read
                }
            }
        }
    }
    // every copy has landed and every product is complete before the memory is given back
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

// Joins the key ranges of a row: one warp per (token row, query head).
template <int D, typename T>
__global__ void __launch_bounds__(256)
paged_chunk_join_kernel(const __grid_constant__ TcShape p, int tile_rows, const uint32_t* __restrict__ q_starts,
                        const uint32_t* __restrict__ seq_lens, const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                        T* __restrict__ out) {
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x;
    const int seq = sequence_of_row(q_starts, p.sh.batch, row);
    if (seq >= p.sh.batch) return;
    const int64_t s = q_starts[seq], e = q_starts[seq + 1], len = seq_lens[seq];
    if (row < s || row >= e || !sequence_ok(p.sh, s, e, len)) return;      // reported by the first kernel
    const int n = int(e - s), token = int(row - s);
    const int chunks = ((int(len) + kTcKeys - 1) / kTcKeys + p.chunk_tiles - 1) / p.chunk_tiles;
    if (chunks == 1) return;                                                                            // written already
    for (int head = blockIdx.y * 8 + warp; head < p.sh.num_q_heads; head += gridDim.y * 8) {
        const int r = token * p.group + head % p.group, last = min((r / tile_rows + 1) * tile_rows, n * p.group) - 1;
        const int limit = int(len) - n + last / p.group + 1;                                            // of the item's last row
        const int used = ((limit + kTcKeys - 1) / kTcKeys + p.chunk_tiles - 1) / p.chunk_tiles;
        const int64_t base = (row * p.sh.num_q_heads + head) * p.max_chunks;
        float m = -INFINITY;
        for (int i = lane; i < used; i += 32) m = fmaxf(m, part_ml[base + i].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float l = 0.0f;
        constexpr int V = D / 32;
        float acc[V];
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.0f;
        for (int i = 0; i < used; ++i) {
            const float2 ml = part_ml[base + i];
            if (ml.x == -INFINITY) continue;           // no visible key in this range, or only scores of -inf
            const float w = ex2(ml.x - m);
            l = fmaf(ml.y, w, l);
            float o[V];
            load_f32<float, V>(part_o + (base + i) * D + lane * V, o);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = fmaf(o[k], fabsf(o[k]) == INFINITY ? 1.0f : w, acc[k]);      // (a weight of zero would make it NaN)
        }
        const float inv = 1.0f / l;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] *= inv;
        store_f32<T, V>(out + (row * p.sh.num_q_heads + head) * D + lane * V, acc);
    }
}
