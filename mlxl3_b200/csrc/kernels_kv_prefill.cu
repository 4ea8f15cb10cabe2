// Attention of many new tokens over a paged key/value cache (prompts, chunks of prompts, draft tokens of wide groups) on the tcgen05
// tensor cores; kernels_kv_attention.cu has the mathematics and takes the sequences of few rows.
//
// A segment is 256 rows of a sequence and key head, its keys come in blocks of 128 (kv_work.cuh).  Per block, tile x (128 rows) of
// the segment: S_x = Q_x K^T (128 x 128, fp32, tensor memory), probabilities P_x = exp2(S_x scale - m) by the 128 threads that own one
// row each, rounded to 16 bits and stored over the half of S_x that was read first, then O_x += P_x V with P_x as the tensor-memory
// operand.  The two tiles share the block's keys and values and take turns: while the tensor cores multiply for one, the other's
// exponentials are computed.  Tensor memory: S_0, S_1, O_0, O_1.
//
// The running maximum m of a row is moved only when a score exceeds it by 2^8 (in log2 units 8): until then O_x and the sum stay in the
// same unit, and probabilities in the range of their type (kv_work.cuh).  When it moves, the row's thread rescales O_x in tensor memory;
// S_x of a block being complete implies that the product before it is, so nothing else has to be waited for.
//
// Four warps bring the data, a tile (a block's keys or values) each in turn, into the 128-byte swizzle that the products read: tensor
// copies of whole pages or parts of pages where every key of the block is visible, else 16 bytes at a time with zeros for what lies
// outside the visible range.  One thread issues the products.  Of a quantised cache those warps load the codes and store them as
// fp16, exactly; the key's scale multiplies its scores and the value's its probability, relative to the row's largest such term
// (kv_work.cuh).  bf16 queries enter those fp16 products multiplied by a power of two of their own.  Every wait is bounded; one that gives up
// sets the status word, all roles run on to the end, and the kernel frees its tensor memory.
//
// Values of blocks that not all rows of a segment see whole are looked through for infinities and NaN by the row threads, between their
// probabilities and the product (why: kernels_kv_attention.cu).  A mixed step with two such blocks a segment took 83 us without and takes 86,
// the prompt 175 and 175; with the look by a warp of its own ahead of the products they took 91 and 178.
//
// What bounds it: for long prompts the chain score product -> softmax -> output product of the two tiles in turn, 3400 cycles a block, of which
// the products need 2864 (a step of K = 16 takes 105 cycles with both operands in shared memory, 74 with the left one in tensor
// memory; the pipe's own time is 64), under the power cap.  4096 tokens, 32 heads of 128 over 8, fp16: 160 us for
// forty calls, 175 us when the power cap has settled.  Segments of one tile leave
// the other idle (their blocks dealt to both pipelines gained 4 %): 16 draft tokens of 8 sequences, five heads to a key head, 8 bits:
// 102 us.
#include "kv_work.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace b200exl3 {

namespace {

constexpr int kManyKeys = 128, kManyTile = 128, kManyRows = 2 * kManyTile;
constexpr int kSoftmaxWarps = 8, kLoadWarps = 4;
constexpr int kManyThreads = 32 * (kSoftmaxWarps + kLoadWarps + 4);   // the last four: one issues the products, two bring queries
// Registers of a thread, of the launch's 128: the row threads hold 64 scores and more, and what spills goes far (shared memory leaves no
// first-level cache).  256 * 160 + 128 * 96 + 128 * 96 <= 512 * 128.
constexpr int kSoftmaxRegisters = 160, kLoadRegisters = 96, kIssueRegisters = 96;
static_assert(8 * kSoftmaxRegisters + 4 * kLoadRegisters + 4 * kIssueRegisters <= 16 * 128, "registers");
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int kQueryWarp = kSoftmaxWarps + kLoadWarps + 1;         // and two bring the queries
constexpr int kManyTable = 512;
// A segment's queries, masks and end in units of a block: us of a prompt of 4096 with 1, 3 and 5 of them 182, 159 and 164, of a mixed step
// 86, 82 and 85.
constexpr int kManyOver = 3;
constexpr uint32_t kScoreCols = 128;               // tensor-memory columns of S_x; P_x lies in their second half

template <int BITS, int D>
struct ManyShape {
    static constexpr int kTileBytes = kManyKeys * D * 2;           // a block's keys or values, as the products read them
    static constexpr int kSlots = D == 128 ? 4 : 6;                // keys and values in flight, alternately
    static constexpr int kQueryBytes = kManyRows * D * 2;
    static constexpr int kStageRow = 80;                           // a row of 32 results on its way out, 64 bytes without bank conflicts
    static constexpr int kStageBytes = kSoftmaxWarps * 32 * kStageRow;
    // blocks whose scales are kept, with codes: [key scales, value scales, their logarithms][128 keys].  One more than in flight: a block's
    // scales are read until the block behind it has its scores, and those free the keys' place of the block that takes the scales' place.
    static constexpr int kScaleBlocks = kSlots / 2 + 1, kScaleFloats = 3 * kManyKeys;
    static constexpr int kScaleBytes = BITS == 16 ? 0 : kScaleBlocks * kScaleFloats * 4;
    static constexpr size_t kSmem = 1024 + kQueryBytes + static_cast<size_t>(kSlots) * kTileBytes + kStageBytes + kScaleBytes;
    static constexpr int kPartFloats = kManyRows * (D + 2);
    static constexpr uint32_t kOutCols = 2 * kScoreCols;           // first column of O_0; O_1 lies D further
};

// D[tmem] (+)= A[smem] . B[smem]
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Values as they lie, [keys][dimensions]: the operand's contiguous axis is the product's N, 64 dimensions (128 bytes, swizzled) by 8
// keys an atom, atoms of further keys 1024 bytes on, the next 64 dimensions `half_bytes` on.
__device__ __forceinline__ uint64_t umma_desc_values(uint32_t smem_byte_addr, uint32_t half_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_byte_addr & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>(half_bytes >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Byte offset of 16-byte chunk c of row r in a tile of `rows` rows: halves of 64 dimensions one after the other, 128-byte swizzle.
__device__ __forceinline__ uint32_t many_at(int rows, int r, int c) {
    return static_cast<uint32_t>((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Two fp32 numbers in one instruction
struct Pair {
    uint64_t v;
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair fma2(Pair a, const Pair& b, const Pair& c) { asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.v) : "l"(b.v), "l"(c.v)); return a; }
__device__ __forceinline__ Pair add2(Pair a, const Pair& b) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v)); return a; }

__device__ __forceinline__ Pair mul2(Pair a, const Pair& b) { asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v)); return a; }
__device__ __forceinline__ void scale2(uint32_t& v0, uint32_t& v1, float f0, float f1) {
    float x0, x1;
    mul2(Pair(__uint_as_float(v0), __uint_as_float(v1)), Pair(f0, f1)).get(x0, x1);
    v0 = __float_as_uint(x0);
    v1 = __float_as_uint(x1);
}
__device__ __forceinline__ void term2(uint32_t& v0, uint32_t& v1, const Pair& by, float a0, float a1) {
    float x0, x1;
    fma2(Pair(__uint_as_float(v0), __uint_as_float(v1)), by, Pair(a0, a1)).get(x0, x1);
    v0 = __float_as_uint(x0);
    v1 = __float_as_uint(x1);
}

// Eight 4-bit codes of a word as fp16 in order: the two of a byte go to the halves of a word, as 1024 + u and 1024 + 16 u
__device__ __forceinline__ void codes4_in_order(uint32_t w, uint32_t (&v)[4]) {
    const uint32_t by = 0x2c003c00u, less_bits = 0xd480e408u;        // 1 and 1/16; -1032 and -72
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t b;
        const uint32_t both = prmt(w, 0u, 0x4040u | i | (i << 8));
        asm("lop3.b32 %0, %1, 0x00f0000f, 0x64006400, 0xea;" : "=r"(b) : "r"(both));       // (both & mask) | bias
        const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&by), *reinterpret_cast<const __half2*>(&less_bits));
        v[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

// What the waits of a CTA share: whether one has given up, and when the products last began a block.
struct ManyState {
    uint32_t failed, clock;
};
__device__ __forceinline__ uint32_t cycles() {
    uint32_t c;
    asm volatile("mov.u32 %0, %%clock;" : "=r"(c));
    return c;
}
// Wait that gives up when the products have stood still for 2^29 cycles (about a third of a second), or at once when another role has given
// up: the second tile's rows wait through all segments of one tile ahead of theirs.  Inlined, since the register split leaves no room
// for a call.
__device__ __forceinline__ void many_wait(uint64_t* bar, uint32_t parity, volatile ManyState* state) {
    if (mbar_try_wait(bar, parity)) return;
    while (!mbar_try_wait_for(bar, parity, 20000)) {
        if (state->failed) return;
        const uint32_t since = state->clock;
        if (static_cast<int32_t>(cycles() - since) > 1 << 29) state->failed = 1;
    }
}

// box_rows: rows of a tensor copy, a power of two that divides the page size, or 0: no tensor copies
template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kManyThreads, 1)
kv_many_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const KvArgs p, const KvAttentionArgs a,
               const int box_rows) {
    using S = ManyShape<BITS, D>;
    using M = std::conditional_t<BITS == 16, T, __half>;          // type of the products
    using Work = KvWork<kManyRows, kManyKeys, kManyOver>;
    using Cursor = KvCursor<kManyRows, kManyKeys, kManyOver>;
    constexpr int kChunks = D / 8;
    constexpr float kUnit = BITS == 16 ? 1.0f : kScaleUnit;      // of the outputs
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ KvTable<kManyTable> s_table;
    __shared__ int64_t s_sum[kManyThreads / 32 + 1];
    // every warp's place, and a row warp's segment at hand: in registers they would push out scores
    __shared__ Cursor s_cursor, s_at[kSoftmaxWarps + kLoadWarps + 3], s_here[kSoftmaxWarps];
    __shared__ __align__(8) uint64_t kv_full[S::kSlots], kv_free[S::kSlots], s_full[2], p_half[2], p_full[2], o_full[2], q_full[2], q_free[2], drained, scales_full[S::kScaleBlocks], raw_full[S::kSlots];
    __shared__ float s_q_scale[2][BITS != 16 && !std::is_same_v<T, __half> ? kManyRows : 1];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int s_last[2];
    __shared__ volatile ManyState s_state;
    // blocks of a row warp's segment at hand with keys that some rows see and others do not: below the first number and from the second on
    __shared__ int2 s_partly[kSoftmaxWarps];
    __shared__ volatile int s_odd;                                // numbers were taken out of such blocks' values

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const Work work(p, a, s_table);
    KvRun run;
    if (!kv_find_run<kManyThreads, 32>(work, s_sum, s_cursor, run)) return;
    unsigned char* const queries = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    unsigned char* const tiles = queries + S::kQueryBytes;
    float* const block_scales = reinterpret_cast<float*>(tiles + S::kSlots * S::kTileBytes + S::kStageBytes);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kSlots; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_free[s], 1); mbar_init(&raw_full[s], 1); }
        for (int x = 0; x < 2; ++x) { mbar_init(&s_full[x], 2); mbar_init(&p_half[x], kManyTile); mbar_init(&p_full[x], kManyTile); mbar_init(&o_full[x], 2); mbar_init(&q_full[x], 1); mbar_init(&q_free[x], 1); }
        mbar_init(&drained, 1);
        for (int i = 0; i < S::kScaleBlocks; ++i) mbar_init(&scales_full[i], 2);
        s_state.failed = 0;
        s_state.clock = cycles();
        s_odd = 0;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == kSoftmaxWarps + kLoadWarps) tmem_alloc(&tmem_base_slot, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base_slot;
    // a warp's cursor moved by all its lanes, to the same place
    auto next_segment = [&](Cursor& c) {
        Cursor next = c;
        const bool ok = next.next_segment(work);
        __syncwarp();
        c = next;
        __syncwarp();
        return ok;
    };

    if (warp < kSoftmaxWarps) {
        // ================= rows: one thread each =================
        more_registers<kSoftmaxRegisters>();
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t scores = tmem + lanes + x * kScoreCols, probs = scores + kScoreCols / 2, outs = tmem + lanes + S::kOutCols + x * D;
        Cursor& at = s_at[warp];
        Cursor& here = s_here[warp];
        at = s_cursor;
        __syncwarp();
        uint32_t s_par = 0, o_par = 0;
        int segment_count = 0;                                    // segments of this tile before
        int block_count = 0, next_count = 0;                      // blocks of the run before this segment's; before the next one's
        bool more = true;                                         // `at` is a segment of this CTA's
        // the cursor at the next segment that has rows of this tile, from where it is
        auto settle = [&]() {
            while (more && x == 1 && work.rows_of(at.seq) - at.tile * kManyRows <= kManyTile) {
                next_count += at.end - at.block;
                more = next_segment(at);
            }
        };
        settle();
        // The values of the block j of the segment at hand.  The look goes over all of them: fewer instructions, whose misses are its time.
        auto look_through = [&](int j) {
            const int vt = 2 * (block_count + j) + 1;
            constexpr int kStep = kManyTile / kChunks;            // a multiple of eight rows: the swizzle is the same
            const int chunk = r % kChunks, row0 = r / kChunks;
            uint32_t at_row = smem_addr(tiles) + vt % S::kSlots * S::kTileBytes + many_at(kManyKeys, row0, chunk);
            many_wait(&kv_full[vt % S::kSlots], (vt / S::kSlots) & 1u, &s_state);
            uint32_t sum = 0, sum2 = 0;
#pragma unroll 1
            for (int k = 0; k < kManyKeys; k += 2 * kStep, at_row += 2 * kStep * 128) {
                uint32_t v[4], w[4];
                shared_load4(at_row, v);
                shared_load4(at_row + kStep * 128, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) { kv_look<T>(sum, v[i]); kv_look<T>(sum2, w[i]); }
            }
            if (__builtin_expect(kv_found(sum | sum2), 0)) {
                s_odd = 1;                                        // before the other tile's threads may find nothing left
                __threadfence_block();
                const int first = here.seg.low + (here.block + j) * kManyKeys;
                const int all0 = work.all_first(here.seq, here.seg) - first, all1 = work.all_end(here.seq, here.seg) - first;
                at_row -= kManyKeys * 128;
#pragma unroll 1
                for (int k = row0; k < kManyKeys; k += kStep, at_row += kStep * 128) {
                    uint32_t v[4];
                    if (k >= all0 && k < all1) continue;          // all rows see it
                    shared_load4(at_row, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = kv_without(v[i], kv_not_finite<T>(v[i]));
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at_row), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
        };
        while (more) {
            {
                block_count = next_count;
                here = at;
                if constexpr (BITS == 16) {
                    if (elect_one()) {
                        const int first = at.seg.low + at.block * kManyKeys;
                        s_partly[warp] = work.several(at.seq) ? make_int2((work.all_first(at.seq, at.seg) - first + kManyKeys - 1) / kManyKeys,
                                                                          (work.all_end(at.seq, at.seg) - first) / kManyKeys)
                                                              : make_int2(0, INT_MAX);
                    }
                }
                __syncwarp();
                const int row = here.tile * kManyRows + x * kManyTile + r, n = here.end - here.block;
                const bool live = row < work.rows_of(here.seq);
                const int position = here.seq.first_pos + row / work.group;
                // visible keys from the first block's first one on
                const int key0 = here.seg.low + here.block * kManyKeys;
                // (no row sees them all, so that nothing is masked for it)
                const int end = live ? kv_seen_end(position, work.capacity) - key0 : INT_MAX, start = (live ? kv_seen_first(position, a.window) : 0) - key0;
                const bool idle = !__any_sync(0xffffffffu, live);              // a warp without rows keeps the barriers and nothing else
                float m = -INFINITY, l = 0.0f, row_scale = a.scale_log2e;
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    const int e = end - j * kManyKeys, b = start - j * kManyKeys;      // visible: columns b .. e - 1
                    many_wait(&s_full[x], s_par, &s_state);
                    s_par ^= 1u;
                    const int kept = (block_count + j) % S::kScaleBlocks;      // the block's scales
                    const float* const key_scales = block_scales + kept * S::kScaleFloats;
                    // written with the queries; two segments' worth, so that the next one's do not overtake a row
                    if (!std::is_same_v<T, M> && j == 0) row_scale = s_q_scale[segment_count & 1][x * kManyTile + r];
                    if constexpr (BITS != 16) many_wait(&scales_full[kept], ((block_count + j) / S::kScaleBlocks) & 1, &s_state);
                    __syncwarp();
                    fence_after();
                    if (j + 1 == n) {
                        next_count = block_count + n;
                        more = next_segment(at);
                        settle();
                    }
                    bool partly = false;                          // some rows of the segment see keys of the block that others do not
                    if constexpr (BITS == 16) {
                        const int2 blocks = s_partly[warp];
                        partly = j < blocks.x || j >= blocks.y;
                    }
                    // the block in two forms, with and without hidden columns: a test between loads and arithmetic costs a sixth of the time
                    auto block = [&](auto with_hidden) {
                    constexpr bool kMasked = decltype(with_hidden)::value;
                    // 64 scores at a time, 32 where scales come on top: longer loops miss the instruction cache
                    constexpr int kWide = BITS == 16 ? 2 : 1, kCols = 32 * kWide;
                    uint32_t v_wide[kWide][32];
                    auto load = [&](int col0) {
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < kWide; ++h) tmem_ld32(scores + col0 + 32 * h, v_wide[h]);
                        tmem_wait_ld();
#pragma unroll
                        for (int h = 0; h < kWide; ++h) {
                        uint32_t (&v)[32] = v_wide[h];
                        const int col = col0 + 32 * h;
                        if constexpr (BITS != 16) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 k = *reinterpret_cast<const float4*>(key_scales + col + i);
                                scale2(v[i], v[i + 1], k.x, k.y);
                                scale2(v[i + 2], v[i + 3], k.z, k.w);
                            }
                        }
                        if constexpr (kMasked) {
                            const int hi = min(max(e - col, 0), 32), lo = min(max(b - col, 0), 32);
                            // bit i: column col + i is visible
                            const uint32_t seen = (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & (lo == 32 ? 0u : 0xffffffffu << lo);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = seen & (1u << i) ? v[i] : 0xff800000u;
                        }
                        }
                    };
                    float top = -INFINITY;
#pragma unroll 1
                    for (int col = 0; col < kManyKeys; col += kCols) {
                        load(col);
                        if constexpr (BITS != 16) {               // terms: scores and the logarithms of the values' scales
                            uint32_t (&v)[32] = v_wide[0];
                            const Pair scales2(row_scale, row_scale);
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 vs_log = *reinterpret_cast<const float4*>(key_scales + 2 * kManyKeys + col + i);
                                term2(v[i], v[i + 1], scales2, vs_log.x, vs_log.y);
                                term2(v[i + 2], v[i + 3], scales2, vs_log.z, vs_log.w);
                            }
                        }
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int h = 0; h < kWide; ++h)
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                t0 = fmaxf(t0, fmaxf(__uint_as_float(v_wide[h][i]), __uint_as_float(v_wide[h][i + 1])));
                                t1 = fmaxf(t1, fmaxf(__uint_as_float(v_wide[h][i + 2]), __uint_as_float(v_wide[h][i + 3])));
                            }
                        top = fmaxf(top, fmaxf(t0, t1));
                    }
                    if constexpr (BITS == 16) top *= row_scale;
                    bool reload = false;
                    const bool moves = top > m + 8.0f;                           // also from -inf
                    if (__any_sync(0xffffffffu, moves)) {
                        const float to = moves ? top : m;
                        const float factor = moves ? exp2_fast(m - to) : 1.0f;
                        m = to;
                        l *= factor;
                        if (j > 0) {
                            reload = true;                            // the outputs' way through the registers
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                __syncwarp();
                                uint32_t o[32];
                                tmem_ld32(outs + c, o);
                                tmem_wait_ld();
                                uint32_t o0[16], o1[16];
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    o0[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                                    o1[i] = __float_as_uint(__uint_as_float(o[16 + i]) * factor);
                                }
                                tmem_st16(outs + c, o0);
                                tmem_st16(outs + c + 16, o1);
                            }
                        }
                    }
                    // from the upper columns down: probabilities go where scores lay that were read before
                    const float shift = m == -INFINITY ? 0.0f : kLift<M> - m;
                    const Pair scales2(row_scale, row_scale), shift2(shift, shift);
                    Pair l2(0.0f, 0.0f), l3(0.0f, 0.0f);
#pragma unroll 1
                    for (int col = kManyKeys - kCols; col >= 0; col -= kCols) {
                        if (kWide == 1 || col + kCols < kManyKeys || reload) load(col);       // 64 at a time: the upper ones are still here
#pragma unroll
                        for (int h = kWide - 1; h >= 0; --h) {
                            const uint32_t (&v)[32] = v_wide[h];
                            uint32_t p2[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                float x0, x1;
                                fma2(Pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scales2, shift2).get(x0, x1);
                                x0 = exp2_fast(x0);
                                x1 = exp2_fast(x1);
                                if (i & 1) l3 = add2(l3, Pair(x0, x1)); else l2 = add2(l2, Pair(x0, x1));
                                if constexpr (BITS != 16) {
                                    const float2 vs = *reinterpret_cast<const float2*>(key_scales + kManyKeys + col + 32 * h + 2 * i);
                                    x0 *= vs.x;
                                    x1 *= vs.y;
                                    if (kMasked) {                // whatever the scale of a hidden key is
                                        if (v[2 * i] == 0xff800000u) x0 = 0.0f;
                                        if (v[2 * i + 1] == 0xff800000u) x1 = 0.0f;
                                    }
                                }
                                p2[i] = KvType<M>::pack(x0, x1);
                            }
                            __syncwarp();
                            tmem_st16(probs + (col + 32 * h) / 2, p2);
                        }
                        if ((col & 32) == 0) {                        // a half is there
                            tmem_wait_st();
                            fence_before();
                            if (BITS != 16 || !partly) mbar_arrive(col == 0 ? &p_full[x] : &p_half[x]);
                        }
                    }
                    l2 = add2(l2, l3);
                    float l0, l1;
                    l2.get(l0, l1);
                    l += l0 + l1;
                    };
                    if (idle) {
                        partly = true;
                    } else if (__any_sync(0xffffffffu, e < kManyKeys || b > 0)) {
                        block(std::true_type{});
                    } else {
                        block(std::false_type{});
                    }
                    if (partly) {
                        // An infinity or NaN among the values of a token would reach the rows that do not see it as 0 times itself.  So the
                        // tile's threads look through such values before the product gets them; what they take out is added at the
                        // segment's end for the rows that see it.
                        if (BITS == 16 && (j < s_partly[warp].x || j >= s_partly[warp].y)) look_through(j);
                        mbar_arrive(&p_half[x]);
                        mbar_arrive(&p_full[x]);
                    }
                }
                // ---- the segment's rows, or this CTA's part of them
                ++segment_count;
                const int64_t first_unit = here.base + kManyOver;
                const int c0 = run.cta_of(first_unit), c1 = run.cta_of(first_unit + here.seg.blocks - 1);
                auto part_of = [&](int c) { return a.parts + (2 * c + (c == c0 ? 1 : 0)) * static_cast<int64_t>(S::kPartFloats); };
                const int pr = x * kManyTile + r;
                const bool whole = c0 == c1;
                // 32 results of the warp's 32 rows at a time go through shared memory, so that four lanes store 64 bytes of a row
                unsigned char* const stage = tiles + S::kSlots * S::kTileBytes + warp * 32 * S::kStageRow;
                T* dst[4];                                        // of the rows that this lane stores a quarter of
                {
                    const int rows_here = work.rows_of(here.seq), lane = threadIdx.x & 31;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int q_row = here.tile * kManyRows + x * kManyTile + (warp & 3) * 32 + i * 8 + lane / 4, q_token = q_row / work.group;
                        dst[i] = q_row < rows_here ? static_cast<T*>(a.out) + (here.seq.first_row + q_token) * a.out_stride +
                                                         static_cast<int64_t>(here.head * work.group + q_row - q_token * work.group) * D + (lane & 3) * 8
                                                   : nullptr;
                    }
                }
                auto store = [&](const float (&v)[32], int c) {   // results c .. c + 31 of this thread's row
                    __syncwarp();
                    const int lane = threadIdx.x & 31;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4*>(stage + lane * S::kStageRow + i * 16) =
                            make_uint4(KvType<T>::pack(v[8 * i], v[8 * i + 1]), KvType<T>::pack(v[8 * i + 2], v[8 * i + 3]),
                                       KvType<T>::pack(v[8 * i + 4], v[8 * i + 5]), KvType<T>::pack(v[8 * i + 6], v[8 * i + 7]));
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (dst[i] != nullptr)
                            *reinterpret_cast<uint4*>(dst[i] + c) = *reinterpret_cast<const uint4*>(stage + (i * 8 + lane / 4) * S::kStageRow + (lane & 3) * 16);
                };
                const float inverse = kv_inverse(l) * kUnit;
                float4* const mine = whole ? nullptr : reinterpret_cast<float4*>(part_of(blockIdx.x)) + pr;      // [four results][row]
                many_wait(&o_full[x], o_par, &s_state);
                o_par ^= 1u;
                __syncwarp();
                fence_after();
                if (BITS == 16 && __builtin_expect(s_odd, 0)) {
                    // values that were taken out of this CTA's blocks come back for the rows that see them (all such: from the first one on
                    // every segment is gone through)
                    const int row = here.tile * kManyRows + x * kManyTile + r, position = here.seq.first_pos + row / work.group;
                    const int low = max(here.seg.low + here.block * kManyKeys, kv_seen_first(position, a.window));
                    const int high = row < work.rows_of(here.seq) ? min(here.seg.low + here.end * kManyKeys, kv_seen_end(position, work.capacity)) : low;
                    const int all0 = work.all_first(here.seq, here.seg), all1 = work.all_end(here.seq, here.seg);
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        __syncwarp();
                        uint32_t o[16];
                        tmem_ld16(outs + c, o);
                        tmem_wait_ld();
#pragma unroll 1
                        for (int key = low; key < high; ++key) {
                            if (key >= all0 && key < all1) key = all1;            // rows of the tile as it was
                            const int64_t place = key < high ? kv_place(p, here.b, key) : -1;
                            if (place < 0) continue;
                            const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.v) +
                                                                                    (place + static_cast<int64_t>(here.head) * p.page_size) * D + c);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const uint32_t w = __ldg(src + i), top_bits = kv_not_finite<T>(w);
                                const float2 f = KvType<T>::unpack(w);
                                if (top_bits & 0x8000u) o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) + f.x);
                                if (top_bits & 0x80000000u) o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) + f.y);
                            }
                        }
                        __syncwarp();
                        tmem_st16(outs + c, o);
                        tmem_wait_st();
                    }
                }
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(outs + c, v);
                    tmem_wait_ld();
                    float f[32];
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]) * inverse;
                        store(f, c);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            __stcg(mine + (c / 4 + i) * kManyRows, make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                                                              __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])));
                    }
                }
                fence_before();
                if (!whole) {
                    reinterpret_cast<float2*>(part_of(blockIdx.x) + kManyRows * D)[pr] = make_float2(m, l);
                    __threadfence();
                    group_sync(1 + x, kManyTile);
                    if (r == 0) {
                        unsigned int* counter = a.arrived + 2 * c0 + x;
                        s_last[x] = atomicAdd(counter, 1u) == static_cast<unsigned int>(c1 - c0);
                        if (s_last[x]) *counter = 0;                              // the next call starts from zero
                    }
                    group_sync(1 + x, kManyTile);
                    if (s_last[x]) {
                        __threadfence();
                        auto weight_of = [&](int c) { return __ldcg(reinterpret_cast<const float2*>(part_of(c) + kManyRows * D) + pr); };
                        float top = -INFINITY, sum = 0.0f;
                        for (int c = c0; c <= c1; ++c) {
                            const float2 ml = weight_of(c);
                            const float to = fmaxf(top, ml.x), safe = to == -INFINITY ? 0.0f : to;
                            sum = sum * exp2_fast(top - safe) + ml.y * exp2_fast(ml.x - safe);
                            top = to;
                        }
                        const float safe = top == -INFINITY ? 0.0f : top, inv = kv_inverse(sum) * kUnit;
#pragma unroll 1
                        for (int d = 0; d < D; d += 32) {
                            float o[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
#pragma unroll 1
                            for (int c = c0; c <= c1; ++c) {
                                const float w = exp2_fast(weight_of(c).x - safe) * inv;
                                const float4* src = reinterpret_cast<const float4*>(part_of(c)) + (d / 4) * kManyRows + pr;
                                float4 f[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) f[i] = __ldcg(src + i * kManyRows);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    o[4 * i] = fmaf(f[i].x, w, o[4 * i]);
                                    o[4 * i + 1] = fmaf(f[i].y, w, o[4 * i + 1]);
                                    o[4 * i + 2] = fmaf(f[i].z, w, o[4 * i + 2]);
                                    o[4 * i + 3] = fmaf(f[i].w, w, o[4 * i + 3]);
                                }
                            }
                            store(o, d);
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        // ================= copies: every warp a tile of its own (even blocks' keys, their values, odd blocks' keys, their values) =================
        fewer_registers<kLoadRegisters>();
        const int w = warp - kSoftmaxWarps, lane = threadIdx.x & 31;
        constexpr int kRowStep = 32 / kChunks;
        const int chunk = lane % kChunks, row0 = lane / kChunks;
        const int parts = box_rows > 0 ? kManyKeys / box_rows : 0;
        const uint32_t tile_base = smem_addr(tiles);
        const char* const pool = static_cast<const char*>(w & 1 ? p.v : p.k) + chunk * 16;
        Cursor& at = s_at[warp];
        at = s_cursor;
        __syncwarp();
        int block = at.block, block_end = at.end;                 // of the segment at hand
        auto step = [&]() {
            if (++block < block_end) return true;
            if (!next_segment(at)) return false;
            block = at.block;
            block_end = at.end;
            return true;
        };
        bool more = w < 2 || step();
        for (int tile = w; more; tile += kLoadWarps) {
            const int slot = tile % S::kSlots, first = at.seg.low + block * kManyKeys;
            // Lane i looks up the i-th part of the block: a tensor copy where every key of it is a token that some row of the sequence
            // sees (and so holds numbers), row by row with zeros where not.
            const int low = kv_seen_first(at.seq.first_pos, a.window);
            const int high = work.any_end(at.seq);
            int64_t from = -1;
            if (lane < parts) {
                const int key = first + lane * box_rows;
                if (key >= low && key + box_rows <= high) from = kv_place(p, at.b, key);
            }
            const uint32_t whole = __ballot_sync(0xffffffffu, from >= 0);
            if (tile >= S::kSlots) {
                many_wait(&kv_free[slot], (tile / S::kSlots - 1) & 1u, &s_state);
                __syncwarp();
            }
            const uint32_t dst = tile_base + slot * S::kTileBytes;
            if constexpr (BITS == 16) {
                if (from >= 0) {
                    const int row = static_cast<int>(from) + at.head * p.page_size;
#pragma unroll
                    for (int h = 0; h < D / 64; ++h)
                        tma_rows(dst + h * kManyKeys * 128 + lane * box_rows * 128, w & 1 ? &v_map : &k_map, h * 128, row, &kv_full[slot]);
                }
                __syncwarp();
                if (__popc(whole) < parts || parts == 0) {
#pragma unroll 1
                    for (int k0 = 0; k0 < kManyKeys; k0 += 32) {  // 32 keys: lane i finds key k0 + i
                        const int key = first + k0 + lane;
                        int64_t place = -1;
                        if (key >= at.seg.key0 && key < at.seg.key1) place = kv_place(p, at.b, key);
                        if (place >= 0) place += static_cast<int64_t>(at.head) * p.page_size;
#pragma unroll
                        for (int i = 0; i < 32 / kRowStep; ++i) {
                            const int r = row0 + i * kRowStep;
                            const int64_t row = __shfl_sync(0xffffffffu, place, r);
                            if (parts == 0 || !(whole >> ((k0 + r) / box_rows) & 1u))
                                copy16_fill(dst + many_at(kManyKeys, k0 + r, chunk), pool + (row < 0 ? 0 : row * (D * 2)), row >= 0);
                        }
                    }
                    copy_commit();
                    copy_wait<0>();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                // the copies' bytes may arrive before they are announced: the phase ends with this arrival at the earliest
                if (lane == 0) mbar_expect_tx(&kv_full[slot], static_cast<uint32_t>(__popc(whole) * box_rows * D * 2));
                __syncwarp();
            } else {
                // Codes come into the end of the tile's own place, row by row what the tensor copies would bring, and are turned into fp16
                // from the first row on: a row's fp16 covers no codes of rows behind it.
                constexpr int kRowBytes = D * BITS / 8, kPieces = kRowBytes / 16;
                const uint32_t raw = dst + S::kTileBytes - kManyKeys * kRowBytes;
                const int kept = (tile >> 1) % S::kScaleBlocks;
                float* const scales = block_scales + kept * S::kScaleFloats + (w & 1) * kManyKeys;
                if (from >= 0) {
                    const int row = static_cast<int>(from) + at.head * p.page_size;
                    tma_rows(raw + lane * box_rows * kRowBytes, w & 1 ? &v_map : &k_map, 0, row, &raw_full[slot]);
                    bulk_copy_g2s(scales + lane * box_rows, (w & 1 ? p.v_scale : p.k_scale) + row, box_rows * 4, &raw_full[slot]);
                }
                __syncwarp();
                if (__popc(whole) < parts || parts == 0) {
#pragma unroll 1
                    for (int k0 = 0; k0 < kManyKeys; k0 += 32) {  // 32 keys: lane i finds key k0 + i
                        if (parts > 0 && box_rows >= 32 && (whole >> (k0 / box_rows) & 1u)) continue;
                        const int key = first + k0 + lane;
                        int64_t place = -1;
                        if (key >= at.seg.key0 && key < at.seg.key1) place = kv_place(p, at.b, key);
                        if (place >= 0) place += static_cast<int64_t>(at.head) * p.page_size;
                        if (parts == 0 || !(whole >> ((k0 + lane) / box_rows) & 1u))
                            scales[k0 + lane] = place >= 0 ? __ldg((w & 1 ? p.v_scale : p.k_scale) + place) : 0.0f;      // hidden keys have none
                        constexpr int kStep = 32 / kPieces;
#pragma unroll
                        for (int i = 0; i < 32 / kStep; ++i) {
                            const int r = i * kStep + lane / kPieces, piece = lane % kPieces;
                            const int64_t row = __shfl_sync(0xffffffffu, place, r);
                            if (parts == 0 || !(whole >> ((k0 + r) / box_rows) & 1u))
                                copy16_fill(raw + tile_at<kPieces, kManyKeys>(k0 + r, piece),
                                            static_cast<const char*>(w & 1 ? p.v : p.k) + (row < 0 ? 0 : row * kRowBytes) + piece * 16, row >= 0);
                        }
                    }
                    copy_commit();
                    copy_wait<0>();
                }
                if (lane == 0) mbar_expect_tx(&raw_full[slot], static_cast<uint32_t>(__popc(whole) * box_rows * (kRowBytes + 4)));
                __syncwarp();
                many_wait(&raw_full[slot], (tile / S::kSlots) & 1u, &s_state);
                __syncwarp();
                if (w & 1) {
#pragma unroll
                    for (int i = lane; i < kManyKeys; i += 32) {
                        const float vs = scales[i] * (1.0f / kScaleUnit);
                        scales[i] = vs;
                        scales[i + kManyKeys] = kv_scale_log(vs);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&scales_full[kept]);
                constexpr int kAtOnce = 32 / kPieces, kTurns = kManyKeys / kAtOnce, kOut = 16 / BITS;      // 16-byte chunks of fp16 out of one of codes
                const int piece = lane % kPieces, sub = lane / kPieces;
#pragma unroll 1
                for (int t0 = 0; t0 < kTurns; t0 += 4) {
                    uint32_t words[4][4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t from_at = raw + tile_at<kPieces, kManyKeys>((t0 + u) * kAtOnce + sub, piece);
                        shared_load4(from_at, words[u]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int row = (t0 + u) * kAtOnce + sub;
                        uint32_t h[4 * kOut];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if constexpr (BITS == 8) {
                                const uint32_t x = words[u][k] ^ 0x80808080u;
                                h[2 * k] = codes8<0, 1>(x);
                                h[2 * k + 1] = codes8<2, 3>(x);
                            } else {
                                uint32_t four[4];
                                codes4_in_order(words[u][k], four);
#pragma unroll
                                for (int i = 0; i < 4; ++i) h[4 * k + i] = four[i];
                            }
                        }
#pragma unroll
                        for (int c = 0; c < kOut; ++c)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + many_at(kManyKeys, row, piece * kOut + c)), "r"(h[4 * c]),
                                         "r"(h[4 * c + 1]), "r"(h[4 * c + 2]), "r"(h[4 * c + 3]) : "memory");
                    }
                    __syncwarp();
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&kv_full[slot]);
            }
            more = step() && step() && !__any_sync(0xffffffffu, s_state.failed != 0);      // then nobody waits for copies any more
        }
    } else {
        fewer_registers<kIssueRegisters>();
        if (warp == kSoftmaxWarps + kLoadWarps && elect_one()) {
        // ================= products =================
        constexpr uint32_t kFormat = std::is_same_v<M, __half> ? 0u : 1u;
        constexpr uint32_t kBase = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((128u >> 4) << 24);
        constexpr uint32_t kScoreDesc = kBase | ((static_cast<uint32_t>(kManyKeys) >> 3) << 17);
        constexpr uint32_t kValueDesc = kBase | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17);    // values: N is the contiguous axis
        const uint64_t q_desc = umma_desc(smem_addr(queries)), k_desc = umma_desc(smem_addr(tiles));
        const uint64_t v_desc = umma_desc_values(smem_addr(tiles), kManyKeys * 128);
        Cursor& at = s_at[warp];
        at = s_cursor;
        int tile = 0;                                             // tiles consumed
        uint32_t p_par[2] = {0, 0}, q_par[2] = {0, 0};
        auto wait_tile = [&](int i) {
            many_wait(&kv_full[i % S::kSlots], (i / S::kSlots) & 1u, &s_state);
            fence_after();
        };
        auto score = [&](int x, int slot) {
            const uint64_t qd = q_desc + x * (S::kQueryBytes / 2 >> 4), kd = k_desc + slot * (S::kTileBytes >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k >> 2) * (kManyTile * 128 >> 4) + (k & 3) * 2;
                umma_f16_ss(tmem + x * kScoreCols, qd + off, kd + off, kScoreDesc, k > 0);
            }
            umma_commit(&s_full[x]);
            mbar_arrive(&s_full[x]);                              // and passes on what this thread has waited for: the rows' scales beside their queries
        };
        auto weigh = [&](int x, int slot, bool accumulate) {
            // the probabilities of the upper keys come first
            const uint64_t vd = v_desc + slot * (S::kTileBytes >> 4);
#pragma unroll
            for (int h = 1; h >= 0; --h) {
                many_wait(h ? &p_half[x] : &p_full[x], p_par[x], &s_state);
                fence_after();
#pragma unroll
                for (int k = h * (kManyKeys / 32); k < (h + 1) * (kManyKeys / 32); ++k)
                    umma_f16_ts(tmem + S::kOutCols + x * D, tmem + x * kScoreCols + kScoreCols / 2 + k * 8, vd + k * (16 * 128 >> 4), kValueDesc,
                                accumulate || h == 0 || k > kManyKeys / 32);
            }
            p_par[x] ^= 1u;
        };
        do {
            const int rows = work.rows_of(at.seq), n = at.end - at.block;
            const bool two = rows - at.tile * kManyRows > kManyTile;
            wait_tile(tile);
            for (int x = 0; x < (two ? 2 : 1); ++x) {
                many_wait(&q_full[x], q_par[x], &s_state);
                q_par[x] ^= 1u;
                fence_after();
                score(x, tile % S::kSlots);
                if (n == 1) umma_commit(&q_free[x]);
            }
            umma_commit(&kv_free[tile % S::kSlots]);
            for (int j = 0; j < n; ++j) {
                const int vt = tile + 1, kt = tile + 2;
                const bool more = j + 1 < n;
                wait_tile(vt);
                weigh(0, vt % S::kSlots, j > 0);
                if (more) {
                    wait_tile(kt);
                    score(0, kt % S::kSlots);
                    if (j + 2 == n) umma_commit(&q_free[0]);
                } else {
                    umma_commit(&o_full[0]);
                    mbar_arrive(&o_full[0]);                    // and passes on what the rows took out
                }
                if (two) {
                    weigh(1, vt % S::kSlots, j > 0);
                    umma_commit(&kv_free[vt % S::kSlots]);
                    if (more) {
                        score(1, kt % S::kSlots);
                        if (j + 2 == n) umma_commit(&q_free[1]);
                    } else {
                        umma_commit(&o_full[1]);
                        mbar_arrive(&o_full[1]);                    // and passes on what the rows took out
                    }
                } else {
                    umma_commit(&kv_free[vt % S::kSlots]);
                }
                if (more) umma_commit(&kv_free[kt % S::kSlots]);
                tile += 2;
                s_state.clock = cycles();
            }
        } while (at.next_segment(work));
        umma_commit(&drained);
        many_wait(&drained, 0, &s_state);
        } else if (warp == kQueryWarp || warp == kQueryWarp + 1) {
            // ================= queries of a tile: neighbouring lanes a row; rows past the last are zeros =================
            const int x = warp - kQueryWarp, lane = threadIdx.x & 31, chunk = lane % kChunks;
            constexpr int kStep = 32 / kChunks;
            const uint32_t dst = smem_addr(queries) + x * (S::kQueryBytes / 2);
            Cursor& at = s_at[warp];
            at = s_cursor;
            __syncwarp();
            int loaded = 0;
            do {
                const int rows = work.rows_of(at.seq);
                if (x == 1 && rows - at.tile * kManyRows <= kManyTile) continue;
                const int row0 = at.tile * kManyRows + x * kManyTile, token0 = row0 / work.group, past = row0 - token0 * work.group;
                const float per_token = 1.0f / static_cast<float>(work.group);
                const T* const base = static_cast<const T*>(a.q) + (at.seq.first_row + token0) * a.q_stride +
                                      static_cast<int64_t>(at.head * work.group) * D + chunk * 8;
                // the products of this tile's segment before have read their queries
                if (loaded > 0) many_wait(&q_free[x], (loaded - 1) & 1, &s_state);
                __syncwarp();
                auto source = [&](int q, bool live) {             // row q of the tile
                    // (past + q) / group: half a row away from where fp32 could round it over an edge
                    const int token = __float2int_rz((static_cast<float>(past + q) + 0.5f) * per_token);
                    return live ? base + token * a.q_stride + (past + q - token * work.group) * D : static_cast<const T*>(a.q);
                };
                if constexpr (std::is_same_v<T, M>) {
#pragma unroll 8
                    for (int q = lane / kChunks; q < kManyTile; q += kStep) {
                        const bool live = row0 + q < rows;
                        copy16_fill(dst + many_at(kManyTile, q, chunk), source(q, live), live);
                    }
                } else {
#pragma unroll 1
                    for (int q0 = lane / kChunks; q0 < kManyTile; q0 += 8 * kStep) {
                        uint4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(source(q0 + i * kStep, row0 + q0 + i * kStep < rows)));
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int q = q0 + i * kStep;
                            uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                            float top = 0.0f;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float2 f = KvType<T>::unpack(w[k]);
                                top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                            }
#pragma unroll
                            for (int d = kChunks / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            const KvPower power(top);
                            const bool live = row0 + q < rows;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float2 f = KvType<T>::unpack(w[k]);
                                w[k] = live ? KvType<M>::pack(f.x * power.down0 * power.down1, f.y * power.down0 * power.down1) : 0u;
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + many_at(kManyTile, q, chunk)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                            if (chunk == 0) s_q_scale[loaded & 1][x * kManyTile + q] = a.scale_log2e * power.up0 * power.up1;
                        }
                    }
                }
                copy_commit();
                copy_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[x]);
                ++loaded;
            } while (next_segment(at));
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    settle_after_failure(s_state.failed != 0);
    if (warp == kSoftmaxWarps + kLoadWarps) {
        __syncwarp();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && s_state.failed) atomicExch(a.error, 8u);
}

template <typename T, int BITS, int D>
cudaError_t launch_many(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
    using S = ManyShape<BITS, D>;
    static PerDeviceOnce attribute;
    if (attribute.needed()) {
        cudaError_t e = cudaFuncSetAttribute(kv_many_kernel<T, BITS, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        attribute.mark();
    }
    CUtensorMap k_map{}, v_map{};
    int box_rows = 0;
    if (!kv_tensor_maps(p, kManyKeys, &k_map, &v_map, &box_rows)) box_rows = 0;
    return launch_dependent(kv_many_kernel<T, BITS, D>, dim3(static_cast<unsigned>(sm_count())), dim3(kManyThreads), S::kSmem, stream, k_map, v_map, p, a,
                            box_rows);
}

}  // namespace

size_t kv_many_workspace_bytes(int head_dim) { return 2 * static_cast<size_t>(sm_count()) * kManyRows * (head_dim + 2) * sizeof(float); }

cudaError_t launch_kv_many(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
#define B200_KV_CASE(T, BITS, D) \
    if (p.bits == BITS && p.head_dim == D) return launch_many<T, BITS, D>(p, a, stream);
#define B200_KV_CASES(T)                                                      \
    B200_KV_CASE(T, 16, 128) B200_KV_CASE(T, 16, 64) B200_KV_CASE(T, 8, 128) \
    B200_KV_CASE(T, 8, 64) B200_KV_CASE(T, 4, 128) B200_KV_CASE(T, 4, 64)
    if (p.dtype == kF16) { B200_KV_CASES(__half) }
    else { B200_KV_CASES(__nv_bfloat16) }
#undef B200_KV_CASES
#undef B200_KV_CASE
    return cudaErrorInvalidValue;
}

}  // namespace b200exl3
