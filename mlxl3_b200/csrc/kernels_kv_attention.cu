// Attention of new tokens over a paged key/value cache: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the tokens j up to its own
// (with a window w: the last w of them).
//
// Work is shared out as kv_work.cuh says, in segments of 8 * NB rows and blocks of 64 keys (128 of codes).
//
// A block: the warps take turns to ask for its keys and values (tensor copies of whole pages or parts of pages, several blocks in flight; row by
// row with zeros at the ends of the visible range and where pages are too small, so that nothing behind a length is ever
// multiplied); four warps take a quarter of the keys each: scores by mma.sync, online softmax in fp32 registers, probabilities rounded to
// 16 bits for the second product.  Loads bound it: what a step of single tokens moves is the cache, once.
// Both products have the keys and values as their left operand and the rows as their right one, whose tiles are 8 wide: a group of four
// query heads leaves half of a tile idle where it would leave three quarters of a left one's 16, and scores, outputs and exponentials
// take half the registers and instructions (long 4-bit contexts 254 -> 208 us; 174 with a third CTA per SM
// and no masks for rows that pad the tile; 64 ragged sequences of bf16 221 us, 98 % of the measured copy rate).
// A row's maximum moves only when a score exceeds it by 2^8, so that outputs are seldom rescaled and the lanes that share a row seldom
// have to agree; what probabilities then reach is in kv_work.cuh.
//
// Codes are multiplied as they are: 8- and 4-bit codes are exact in fp16, and so is what the tensor cores add up in fp32; the key's
// scale multiplies its scores, the value's its probability, relative to the largest such term of the row (kv_work.cuh).  bf16 queries
// enter fp16 multiplied by a power of two of their own (exact but for what lies 2^-24 below the row's largest).
#include "kv_work.cuh"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace b200exl3 {

namespace {

constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps;
constexpr int kFewTable = 128;
// A segment's queries, its end and its part of a join in units of a block: us of 64 ragged sequences with 0, 1, 3, 5 and 8 of them 262,
// 243, 225, 221 and 222, of 16 long ones in 4 bits 181, 178, 178, 174 and 175.
constexpr int kFewOver = 5;

template <int BITS, int D, int NB>
struct FewShape {
    static constexpr int kCtas = BITS == 4 && NB == 1 ? 3 : 2;      // per SM
    static constexpr int kKeys = BITS == 16 ? 64 : 128;            // of a block
    static constexpr int kWarpKeys = kKeys / kFewWarps;            // they share the rows and take different keys
    static constexpr int kStepKeys = std::min(kWarpKeys, 32);      // of a warp's step
    static constexpr int kRows = 8 * NB;
    static constexpr int kRowBytes = D * BITS / 8, kChunks = kRowBytes / 16;
    static constexpr int kTileBytes = kKeys * kRowBytes;
    static constexpr int kScaleBytes = BITS == 16 ? 0 : 2 * kKeys * 4;
    static constexpr int kStageBytes = (2 * kTileBytes + kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kMergeBytes = kFewWarps * kRows * D * 4;  // outputs of the warps, joined in the block's own place where they fit
    static constexpr bool kMergeInStage = kMergeBytes <= kStageBytes;
    static constexpr int kOwnMergeBytes = kMergeInStage ? 0 : kMergeBytes;
    static constexpr int kStages = std::min(6, (222 * 1024 / kCtas - 2 * 1024 - kOwnMergeBytes) / kStageBytes);
    static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStageBytes + kOwnMergeBytes;
    static constexpr int kPartFloats = kRows * (D + 2);
    static_assert(kStages >= 3, "copies in flight");
};

// announces that this thread's copies so far have landed
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename M>
__device__ __forceinline__ void mma_rows(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<M, __half>) {
        mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The same for chunk c + of, c even and of 0 or 1, from the place of chunk `of`: the swizzle is an exclusive or.
template <int CHUNKS, int KEYS>
__device__ __forceinline__ uint32_t tile_next(uint32_t at, int c) {
    constexpr int kPiece = CHUNKS >= 8 ? 8 : CHUNKS;
    return (at ^ static_cast<uint32_t>((c % kPiece) << 4)) + static_cast<uint32_t>(c / kPiece * KEYS * kPiece * 16);
}

// Matrices of 8 x 8 numbers of 16 bits, held as the products hold them, turned over
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

// box_rows: rows of a tensor copy, a power of two that divides the page size, or 0: no tensor copies.  SEVERAL: sequences may have more
// than one row, and so rows that do not see what others do.
template <typename T, int BITS, int D, int NB, bool SEVERAL>
__global__ void __launch_bounds__(kFewThreads, FewShape<BITS, D, NB>::kCtas)
kv_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const KvArgs p, const KvAttentionArgs a,
              const int box_rows) {
    using S = FewShape<BITS, D, NB>;
    using M = std::conditional_t<BITS == 16, T, __half>;          // type of the products
    using Work = KvWork<S::kRows, S::kKeys, kFewOver>;
    using Cursor = KvCursor<S::kRows, S::kKeys, kFewOver>;
    constexpr int kTiles = D / 16, kSteps = D / 16;               // tiles of the output, steps of the first product
    constexpr int kSub = S::kStepKeys / 16;                       // tiles of keys of a warp's step
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ int64_t s_sum[kFewThreads + 1];
    __shared__ KvTable<kFewTable> s_table;
    __shared__ Cursor s_cursor, s_put[kFewWarps], s_get[kFewWarps];
    __shared__ float2 s_ml[kFewWarps][S::kRows];
    __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages];
    __shared__ bool s_last;
    __shared__ volatile int s_failed, s_odd;                      // s_odd: numbers were taken out of values
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    if (threadIdx.x == 0) {
        // a block is there when its tensor copies are (lane 0 says how many bytes) and every lane's own copies
        for (int i = 0; i < S::kStages; ++i) { mbar_init(&full[i], 33); mbar_init(&empty[i], kFewWarps); }
        s_failed = 0;
        s_odd = 0;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const Work work(p, a, s_table);
    KvRun run;
    if (!kv_find_run<kFewThreads, 1>(work, s_sum, s_cursor, run)) return;
    const uint32_t base = smem_addr(smem);

    // ---- copies ------------------------------------------------------------------------------------------------------
    const int parts = box_rows > 0 ? S::kKeys / box_rows : 0;
    // a warp asks for the block at `at`; where the place was used before, once all warps are through with it
    auto copy_block = [&](const Cursor& at, int block, int stage, bool wait, uint32_t parity) {
        const int chunk = lane % S::kChunks, row0 = lane / S::kChunks;
        constexpr int kRowStep = 32 / S::kChunks;
        const int first = at.seg.low + block * S::kKeys;
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
        if (wait) qmm_wait(&empty[stage], parity, &s_failed);
        __syncwarp();
        const uint32_t dst = base + stage * S::kStageBytes;
        if (from >= 0) {
            const int row = static_cast<int>(from) + at.head * p.page_size;
#pragma unroll
            for (int c = 0; c < S::kRowBytes; c += 128) {
                constexpr int kWidth = S::kRowBytes < 128 ? S::kRowBytes : 128;
                const uint32_t to = dst + c * S::kKeys + lane * box_rows * kWidth;
                tma_rows(to, &k_map, c, row, &full[stage]);
                tma_rows(to + S::kTileBytes, &v_map, c, row, &full[stage]);
            }
            if constexpr (BITS != 16) {
                unsigned char* const to = smem + stage * S::kStageBytes + 2 * S::kTileBytes + lane * box_rows * 4;
                bulk_copy_g2s(to, p.k_scale + row, box_rows * 4, &full[stage]);
                bulk_copy_g2s(to + S::kKeys * 4, p.v_scale + row, box_rows * 4, &full[stage]);
            }
        }
        __syncwarp();
        if (parts == 0 || __popc(whole) < parts) {
            const int64_t head = static_cast<int64_t>(at.head) * p.page_size;
#pragma unroll 1
            for (int k0 = 0; k0 < S::kKeys; k0 += 32) {       // 32 keys: lane i finds key k0 + i
                const int key = first + k0 + lane;
                int64_t place = -1;
                if (key >= at.seg.key0 && key < at.seg.key1) place = kv_place(p, at.b, key);
                if (place >= 0) place += head;
                if (BITS != 16 && (parts == 0 || !(whole >> ((k0 + lane) / box_rows) & 1u))) {
                    const uint32_t to = dst + 2 * S::kTileBytes + (k0 + lane) * 4;
                    copy4_fill(to, p.k_scale + (place < 0 ? 0 : place), place >= 0);
                    copy4_fill(to + S::kKeys * 4, p.v_scale + (place < 0 ? 0 : place), place >= 0);
                }
#pragma unroll
                for (int i = 0; i < 32 / kRowStep; ++i) {
                    const int r = row0 + i * kRowStep;
                    const int64_t row = __shfl_sync(0xffffffffu, place, r);
                    if (parts == 0 || !(whole >> ((k0 + r) / box_rows) & 1u)) {
                        const uint32_t to = dst + tile_at<S::kChunks, S::kKeys>(k0 + r, chunk);
                        const int64_t src = (row < 0 ? 0 : row) * S::kRowBytes + chunk * 16;
                        copy16_fill(to, static_cast<const char*>(p.k) + src, row >= 0);
                        copy16_fill(to + S::kTileBytes, static_cast<const char*>(p.v) + src, row >= 0);
                    }
                }
            }
        }
        copy_arrive(&full[stage]);
        if (lane == 0) mbar_expect_tx(&full[stage], static_cast<uint32_t>(__popc(whole) * box_rows * 2 * (S::kRowBytes + (BITS == 16 ? 0 : 4))));
        __syncwarp();
    };
    // Copies (put) run ahead of the products (get).  Every warp keeps both places for itself in shared memory and in registers only which
    // blocks of the segment are left.
    Cursor& put = s_put[warp];
    Cursor& get = s_get[warp];
    auto next_segment = [&](Cursor& c) {
        Cursor next = c;
        const bool ok = next.next_segment(work);
        __syncwarp();
        c = next;                                                 // the same from all lanes
        __syncwarp();
        return ok;
    };
    put = s_cursor;
    get = s_cursor;
    __syncwarp();
    int put_block = put.block, put_end = put.end;
    bool more = true;                                             // put stands at a block
    auto step_put = [&]() {
        if (++put_block < put_end) return true;
        if (!next_segment(put)) return false;
        put_block = put.block;
        put_end = put.end;
        return true;
    };
    for (int i = 0; i < S::kStages - 1 && more; ++i) {
        if (i % kFewWarps == warp) copy_block(put, put_block, i, false, 0);
        more = step_put();
    }

    // ---- state of a segment ---------------------------------------------------------------------------------------------
    // A lane holds the queries of row 8 b + g; scores, sums and outputs of rows 8 b + 2 t and the next (e = 0, 1).
    uint32_t q[NB][kSteps][2];
    float out[NB][kTiles][4], m[NB][2], l[NB][2], row_scale[NB][2];
    int key_end[NB][2], key_start[NB][2];                         // keys that a row sees; no row sees them all, so that nothing is masked for it
    auto begin = [&]() {
        const int rows = work.rows_of(get.seq);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int row0 = get.tile * S::kRows + 8 * b;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = row0 + 2 * t + e;
                const int position = get.seq.first_pos + r / work.group;
                key_end[b][e] = r < rows ? kv_seen_end(position, work.capacity) : INT_MAX;
                key_start[b][e] = r < rows ? kv_seen_first(position, a.window) : 0;
                m[b][e] = -INFINITY;
                l[b][e] = 0.0f;
                row_scale[b][e] = a.scale_log2e;
            }
#pragma unroll
            for (int i = 0; i < kTiles; ++i) out[b][i][0] = out[b][i][1] = out[b][i][2] = out[b][i][3] = 0.0f;
            const int r = row0 + g, token = r / work.group;
            const T* const src = static_cast<const T*>(a.q) + (get.seq.first_row + token) * a.q_stride +
                                 static_cast<int64_t>(get.head * work.group + r - token * work.group) * D;
            // the order of the dimensions within a step is the one the keys come in
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int w = 0; w < 2; ++w) {                     // places 2t, 2t + 1 and 2t + 8, 2t + 9 of the step
                    uint32_t v = 0;
                    if (r < rows) {
                        if constexpr (BITS == 16) v = *reinterpret_cast<const uint32_t*>(src + s * 16 + 2 * t + 8 * w);
                        else if constexpr (BITS == 8) v = *reinterpret_cast<const uint32_t*>(src + s * 16 + 4 * t + 2 * w);
                        else {
                            const uint16_t* e = reinterpret_cast<const uint16_t*>(src) + (s >> 1) * 32 + 8 * t + 2 * (s & 1) + w;
                            v = e[0] | static_cast<uint32_t>(e[4]) << 16;
                        }
                    }
                    q[b][s][w] = v;
                }
            if constexpr (!std::is_same_v<T, M>) {
                // bf16 rows enter fp16 products: scaled by the power of two that brings the row's largest to [1, 2)
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float2 f = KvType<T>::unpack(q[b][s][w]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const KvPower power(top);
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float2 f = KvType<T>::unpack(q[b][s][w]);
                        q[b][s][w] = KvType<M>::pack(f.x * power.down0 * power.down1, f.y * power.down0 * power.down1);
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    row_scale[b][e] = row_scale[b][e] * __shfl_sync(0xffffffffu, power.up0, (2 * t + e) * 4) * __shfl_sync(0xffffffffu, power.up1, (2 * t + e) * 4);
            }
        }
    };

    // An infinity or NaN among the values of a token would reach the rows that do not see it as 0 times itself: it is taken out of the
    // warp's keys before the product, and added at the segment's end for the rows that see it.
    auto look_through = [&](uint32_t values, int wrow, int block_key) {
        constexpr int kStep = 32 / S::kChunks;
        const int chunk = lane % S::kChunks, row0 = lane / S::kChunks;
        uint32_t sum = 0;
#pragma unroll 4
        for (int r = row0; r < S::kStepKeys; r += kStep) {
            uint32_t w[4];
            shared_load4(values + tile_at<S::kChunks, S::kKeys>(wrow + r, chunk), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) kv_look<T>(sum, w[j]);
        }
        if (__builtin_expect(!__any_sync(0xffffffffu, kv_found(sum)), 1)) return;
        const int all0 = work.all_first(get.seq, get.seg) - block_key, all1 = work.all_end(get.seq, get.seg) - block_key;
#pragma unroll 1
        for (int r = wrow + row0; r < wrow + S::kStepKeys; r += kStep) {
            if (r >= all0 && r < all1) continue;
            const uint32_t place = values + tile_at<S::kChunks, S::kKeys>(r, chunk);
            uint32_t w[4];
            shared_load4(place, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kv_without(w[j], kv_not_finite<T>(w[j]));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        s_odd = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the place goes back to the tensor copies
        __syncwarp();
    };

    // ---- a step of a warp's keys ----------------------------------------------------------------------------------------
    auto multiply = [&](int stage, int wrow, int block_key) {
        const uint32_t keys = base + stage * S::kStageBytes, values = keys + S::kTileBytes;
        // matrices of a load: (octet of keys, chunk) = (0, 0) (1, 0) (0, 1) (1, 1), or (0, 0) (0, 1) (1, 0) (1, 1)
        const int row_a = (lane & 7) + ((lane >> 3) & 1) * 8, chunk_a = lane >> 4, row_b = (lane & 7) + (lane >> 4) * 8, chunk_b = (lane >> 3) & 1;
        float s[kSub][NB][4];                                     // keys g and g + 8, rows 2t and 2t + 1
#pragma unroll
        for (int k = 0; k < kSub; ++k)
#pragma unroll
            for (int b = 0; b < NB; ++b) s[k][b][0] = s[k][b][1] = s[k][b][2] = s[k][b][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; c += 2)
#pragma unroll
            for (int k = 0; k < kSub; ++k) {
                uint32_t r[4];
                ldmatrix4(tile_next<S::kChunks, S::kKeys>(keys + tile_at<S::kChunks, S::kKeys>(wrow + k * 16 + row_a, chunk_a), c), r);
                auto product = [&](int step, const uint32_t (&v)[4]) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma_rows<M>(s[k][b], v, q[b][step][0], q[b][step][1]);
                };
                if constexpr (BITS == 16) {
                    product(c / 2, r);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (BITS == 8) {
                            const uint32_t w0 = r[2 * j] ^ 0x80808080u, w1 = r[2 * j + 1] ^ 0x80808080u;
                            product(c + j, {codes8<0, 1>(w0), codes8<0, 1>(w1), codes8<2, 3>(w0), codes8<2, 3>(w1)});
                        } else {
                            const uint32_t w0 = r[2 * j], w1 = r[2 * j + 1];
                            product(2 * (c + j), {codes4<0>(w0), codes4<0>(w1), codes4<1>(w0), codes4<1>(w1)});
                            product(2 * (c + j) + 1, {codes4<2>(w0), codes4<2>(w1), codes4<3>(w0), codes4<3>(w1)});
                        }
                    }
                }
            }
        const float* scales = reinterpret_cast<const float*>(smem + stage * S::kStageBytes + 2 * S::kTileBytes) + wrow + g;
        float vs[kSub][2], vs_log[kSub][2];
        bool rescale = false;
        float factor[NB][2];                                      // of the outputs so far
#pragma unroll
        for (int b = 0; b < NB; ++b) factor[b][0] = factor[b][1] = 1.0f;
        if constexpr (BITS != 16) {
#pragma unroll
            for (int k = 0; k < kSub; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float ks = scales[k * 16 + 8 * h];
                    vs[k][h] = scales[S::kKeys + k * 16 + 8 * h] * (1.0f / kScaleUnit);
                    vs_log[k][h] = kv_scale_log(vs[k][h]);
                    if (SEVERAL) {                                // a scale that is not finite makes the scores of its key NaN, for the rows that see it
                        ks = fmaf(vs[k][h], 0.0f, ks);
                        vs[k][h] = fminf(vs[k][h], FLT_MAX / kScaleUnit);
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) { s[k][b][2 * h] *= ks; s[k][b][2 * h + 1] *= ks; }
                }
        }
        // masks, maximum, probabilities
        const int first = block_key + wrow + g;
        bool hidden = false;                                      // some row does not see some key; the same for all lanes
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int end = key_end[b][e] - first, start = key_start[b][e] - first;
                if (__any_sync(0xffffffffu, end < S::kStepKeys - 7 || start > 0)) {
                    hidden = true;
#pragma unroll
                    for (int k = 0; k < kSub; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (k * 16 + 8 * h >= end || k * 16 + 8 * h < start) s[k][b][2 * h + e] = -INFINITY;
                }
                float top = -INFINITY;
                if constexpr (BITS == 16) {
#pragma unroll
                    for (int k = 0; k < kSub; ++k) top = fmaxf(top, fmaxf(s[k][b][e], s[k][b][2 + e]));
                    top *= row_scale[b][e];
                } else {
#pragma unroll
                    for (int k = 0; k < kSub; ++k)
                        top = fmaxf(top, fmaxf(fmaf(s[k][b][e], row_scale[b][e], vs_log[k][0]), fmaf(s[k][b][2 + e], row_scale[b][e], vs_log[k][1])));
                }
                if (__any_sync(0xffffffffu, top > m[b][e] + 8.0f)) {              // also from -inf
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    if (top > m[b][e]) {                          // the same for all lanes of the row
                        const float c = exp2_fast(m[b][e] - top);
                        m[b][e] = top;
                        l[b][e] *= c;
                        factor[b][e] *= c;
                    }
                    rescale = true;
                }
            }
        if (rescale) {                                            // the same for all lanes
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    out[b][i][0] *= factor[b][0]; out[b][i][1] *= factor[b][1]; out[b][i][2] *= factor[b][0]; out[b][i][3] *= factor[b][1];
                }
        }
        if constexpr (BITS == 16)
            if (SEVERAL && hidden && work.several(get.seq)) look_through(values, wrow, block_key);
        uint32_t pr[kSub][NB][2];                                 // probabilities as the right operand: keys 2t, 2t + 1 (+ 8) of row g
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float shift[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) shift[e] = m[b][e] == -INFINITY ? 0.0f : kLift<M> - m[b][e];        // a row that saw nothing yet
#pragma unroll
            for (int k = 0; k < kSub; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[e] = exp2_fast(fmaf(s[k][b][2 * h + e], row_scale[b][e], shift[e]));
                        l[b][e] += x[e];
                        if constexpr (BITS != 16) x[e] *= vs[k][h];
                    }
                    pr[k][b][h] = transposed(KvType<M>::pack(x[0], x[1]));
                }
        }
        // values times probabilities
#pragma unroll
        for (int k = 0; k < kSub; ++k)
#pragma unroll
            for (int c = 0; c < S::kChunks; c += 2) {
                uint32_t r[4];
                auto product = [&](int tile, const uint32_t (&v)[4]) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma_rows<M>(out[b][tile], v, pr[k][b][0], pr[k][b][1]);
                };
                if constexpr (BITS == 16) {
                    ldmatrix4_trans(tile_next<S::kChunks, S::kKeys>(values + tile_at<S::kChunks, S::kKeys>(wrow + k * 16 + row_b, chunk_b), c), r);
                    product(c / 2, r);
                } else {
                    ldmatrix4_trans(tile_next<S::kChunks, S::kKeys>(values + tile_at<S::kChunks, S::kKeys>(wrow + k * 16 + row_a, chunk_a), c), r);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (BITS == 8) {
                            const uint32_t w0 = r[2 * j] ^ 0x80808080u, w1 = r[2 * j + 1] ^ 0x80808080u;
                            product(c + j, {codes8<0, 2>(w0), codes8<1, 3>(w0), codes8<0, 2>(w1), codes8<1, 3>(w1)});
                        } else {
                            const uint32_t w0 = r[2 * j], w1 = r[2 * j + 1];
                            product(2 * (c + j), {codes4<0>(w0), codes4<1>(w0), codes4<0>(w1), codes4<1>(w1)});
                            product(2 * (c + j) + 1, {codes4<2>(w0), codes4<3>(w0), codes4<2>(w1), codes4<3>(w1)});
                        }
                    }
                }
            }
    };
    // dimension of out[.][i][2 h + e]: where the values' chunks put it
    auto dim_of = [&](int i, int h) {
        if constexpr (BITS == 16) return i * 16 + 8 * h + g;
        else if constexpr (BITS == 8) return i * 16 + 2 * g + h;
        else return (i >> 1) * 32 + 4 * g + 2 * (i & 1) + h;
    };

    // ---- end of a segment, or of this CTA's part of it ----------------------------------------------------------------
    // The warps' outputs of the rows that there are go through shared memory; then a warp at a time holds a row, joins what the warps
    // made of their keys and stores it, or this CTA's part of it.
    constexpr int kLaneDims = D / 32;
    auto store_row = [&](int r, const float (&v)[kLaneDims]) {            // row r of the segment's sequence; this lane's dimensions
        const int token = r / work.group;
        T* dst = static_cast<T*>(a.out) + (get.seq.first_row + token) * a.out_stride +
                 static_cast<int64_t>(get.head * work.group + r - token * work.group) * D + lane * kLaneDims;
#pragma unroll
        for (int e = 0; e < kLaneDims; e += 2) reinterpret_cast<uint32_t*>(dst)[e / 2] = KvType<T>::pack(v[e], v[e + 1]);
    };
    auto load_row = [&](const float* src, float (&v)[kLaneDims]) {
        if constexpr (kLaneDims == 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(src) + lane);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const float2 f = __ldcg(reinterpret_cast<const float2*>(src) + lane);
            v[0] = f.x; v[1] = f.y;
        }
    };
    // what was taken out of this CTA's blocks, where row r of the segment's sequence sees it (from the first such number on all segments
    // are gone through)
    auto add_odd = [&](int r, float (&o)[kLaneDims]) {
        const int position = get.seq.first_pos + r / work.group, all0 = work.all_first(get.seq, get.seg), all1 = work.all_end(get.seq, get.seg);
        const int end = min(get.seg.low + get.end * S::kKeys, kv_seen_end(position, work.capacity));
#pragma unroll 1
        for (int key = max(get.seg.low + get.block * S::kKeys, kv_seen_first(position, a.window)); key < end; ++key) {
            if (key >= all0 && key < all1) key = all1;
            const int64_t place = key < end ? kv_place(p, get.b, key) : -1;
            if (place < 0) continue;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.v) + (place + static_cast<int64_t>(get.head) * p.page_size) * D) + lane * (kLaneDims / 2);
#pragma unroll
            for (int e = 0; e < kLaneDims; e += 2) {
                const uint32_t w = __ldg(src + e / 2), top_bits = kv_not_finite<T>(w);
                const float2 f = KvType<T>::unpack(w);
                if (top_bits & 0x8000u) o[e] += f.x;
                if (top_bits & 0x80000000u) o[e + 1] += f.y;
            }
        }
    };
    auto finish = [&](int stage) {
        float* const merge = reinterpret_cast<float*>(smem + (S::kMergeInStage ? stage : S::kStages) * S::kStageBytes);      // [row][warp of its keys][dimension]
        const int tile0 = get.tile * S::kRows, rows_here = min(S::kRows, work.rows_of(get.seq) - tile0);
        group_sync(1, 32 * kFewWarps);                            // every warp is through with the block
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], d);
                const int r = 8 * b + 2 * t + e;
                if (r < rows_here) {
                    if (g == 0) s_ml[warp][r] = make_float2(m[b][e], l[b][e]);
                    float* dst = merge + (r * kFewWarps + warp) * D;
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) dst[dim_of(i, h)] = out[b][i][2 * h + e];
                }
            }
        group_sync(1, 32 * kFewWarps);
        const int64_t first_unit = get.base + kFewOver;
        const int c0 = run.cta_of(first_unit), c1 = run.cta_of(first_unit + get.seg.blocks - 1);      // CTAs that hold its first and last block
        // a CTA's part: its first place for a segment that began before its run, else the second
        auto part_of = [&](int c) { return a.parts + (2 * c + (c == c0 ? 1 : 0)) * static_cast<int64_t>(S::kPartFloats); };
#pragma unroll 1
        for (int r = warp; r < rows_here; r += kFewWarps) {
            float top = -INFINITY, sum = 0.0f, o[kLaneDims];
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, s_ml[w][r].x);
            const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int e = 0; e < kLaneDims; ++e) o[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float2 ml = s_ml[w][r];
                const float c = exp2_fast(ml.x - safe);
                sum = fmaf(ml.y, c, sum);
                const float* src = merge + (r * kFewWarps + w) * D + lane * kLaneDims;
#pragma unroll
                for (int e = 0; e < kLaneDims; ++e) o[e] = fmaf(src[e], c, o[e]);
            }
            if constexpr (BITS == 16)
                if (SEVERAL && __builtin_expect(s_odd, 0)) add_odd(tile0 + r, o);
            if (c0 == c1) {
                const float inverse = kv_inverse(sum) * (BITS == 16 ? 1.0f : kScaleUnit);
#pragma unroll
                for (int e = 0; e < kLaneDims; ++e) o[e] *= inverse;
                store_row(tile0 + r, o);
            } else {
                float* part = part_of(blockIdx.x);
                if (lane == 0) reinterpret_cast<float2*>(part + S::kRows * D)[r] = make_float2(top, sum);
#pragma unroll
                for (int e = 0; e < kLaneDims; ++e) part[r * D + lane * kLaneDims + e] = o[e];
            }
        }
        if (c0 != c1) {
            __threadfence();
            group_sync(1, 32 * kFewWarps);
            if (threadIdx.x == 0) {
                const unsigned int before = atomicAdd(a.arrived + c0, 1u);
                s_last = before == static_cast<unsigned int>(c1 - c0);
                if (s_last) a.arrived[c0] = 0;                    // the next call starts from zero
            }
            group_sync(1, 32 * kFewWarps);
            if (s_last) {
                __threadfence();
                // a warp's lanes weigh the parts, then every lane adds its dimensions over the parts in order
                const int parts = c1 - c0 + 1;
#pragma unroll 1
                for (int r = warp; r < rows_here; r += kFewWarps) {
                    auto weight_of = [&](int i) { return __ldcg(reinterpret_cast<const float2*>(part_of(c0 + i) + S::kRows * D) + r); };
                    float top = -INFINITY;
                    for (int i = lane; i < parts; i += 32) top = fmaxf(top, weight_of(i).x);
#pragma unroll
                    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float safe = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f, o[kLaneDims];
#pragma unroll
                    for (int e = 0; e < kLaneDims; ++e) o[e] = 0.0f;
                    for (int i0 = 0; i0 < parts; i0 += 32) {
                        float2 ml = make_float2(-INFINITY, 0.0f);
                        if (i0 + lane < parts) ml = weight_of(i0 + lane);
                        const float c = exp2_fast(ml.x - safe);
                        sum += c * ml.y;
                        // sixteen parts on their way at a time; what is none counts for nothing
                        for (int j = i0; j < min(i0 + 32, parts); j += 16) {
                            float v[16][kLaneDims];
#pragma unroll
                            for (int i = 0; i < 16; ++i) load_row(part_of(c0 + min(j + i, parts - 1)) + r * D, v[i]);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float w = __shfl_sync(0xffffffffu, c, (j - i0 + i) & 31);
#pragma unroll
                                for (int e = 0; e < kLaneDims; ++e) o[e] = fmaf(v[i][e], j + i < parts ? w : 0.0f, o[e]);
                            }
                        }
                    }
#pragma unroll
                    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    const float inverse = kv_inverse(sum) * (BITS == 16 ? 1.0f : kScaleUnit);
#pragma unroll
                    for (int e = 0; e < kLaneDims; ++e) o[e] *= inverse;
                    store_row(tile0 + r, o);
                }
            }
        }
        // the block's place goes back to the tensor copies
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        group_sync(1, 32 * kFewWarps);
    };

    // ---- the run ------------------------------------------------------------------------------------------------------
    begin();
    int block_key = get.seg.low + get.block * S::kKeys, left = get.end - get.block;      // first key of the block; blocks of the segment
    uint32_t parity = 0;
    for (int stage = 0, turn = S::kStages - 1;; ++turn) {
        if (more) {
            // into the place of the block before: used by it in the round before this one where stage is 0
            const bool used = turn >= S::kStages;
            const int to = stage == 0 ? S::kStages - 1 : stage - 1;
            if (turn % kFewWarps == warp) copy_block(put, put_block, to, used, stage == 0 ? parity ^ 1u : parity);
            more = step_put();
        }
        qmm_wait(&full[stage], parity, &s_failed);
        __syncwarp();
#pragma unroll 1
        for (int k = 0; k < S::kWarpKeys; k += S::kStepKeys) multiply(stage, warp * S::kWarpKeys + k, block_key);
        block_key += S::kKeys;
        const bool end = --left == 0;
        if (end) finish(stage);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (end) {
            if (!next_segment(get)) break;
            begin();
            block_key = get.seg.low + get.block * S::kKeys;
            left = get.end - get.block;
        }
        if (++stage == S::kStages) { stage = 0; parity ^= 1u; }
    }
    __syncthreads();
    settle_after_failure(s_failed != 0);
    if (threadIdx.x == 0 && s_failed) atomicExch(a.error, 8u);
}

template <typename T, int BITS, int D, int NB, bool SEVERAL>
cudaError_t launch_few_rows(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
    using S = FewShape<BITS, D, NB>;
    static PerDeviceOnce attribute;
    if (attribute.needed()) {
        cudaError_t e = cudaFuncSetAttribute(kv_few_kernel<T, BITS, D, NB, SEVERAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        attribute.mark();
    }
    CUtensorMap k_map{}, v_map{};
    int box_rows = 0;
    if (!kv_tensor_maps(p, S::kKeys, &k_map, &v_map, &box_rows)) box_rows = 0;
    return launch_dependent(kv_few_kernel<T, BITS, D, NB, SEVERAL>, dim3(static_cast<unsigned>(S::kCtas * sm_count())), dim3(kFewThreads), S::kSmem, stream,
                            k_map, v_map, p, a, box_rows);
}

template <typename T, int BITS, int D, int NB>
cudaError_t launch_few(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
    return a.max_new > 1 ? launch_few_rows<T, BITS, D, NB, true>(p, a, stream) : launch_few_rows<T, BITS, D, NB, false>(p, a, stream);
}

// Up to this many rows per key head the few-row kernel takes a sequence.
constexpr int kFewRows = 16;

template <typename T, int BITS, int D>
cudaError_t launch_attention(const KvArgs& p, KvAttentionArgs a, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.max_new) * (a.heads / p.kv_heads);
    a.least_rows = 1;
    a.most_rows = INT32_MAX;
    if (rows <= 8) return launch_few<T, BITS, D, 1>(p, a, stream);
    if (rows <= kFewRows) return launch_few<T, BITS, D, 2>(p, a, stream);
    if (p.batch > 1) {                                            // sequences of few rows among the others
        a.most_rows = kFewRows;
        const cudaError_t e = launch_few<T, BITS, D, 2>(p, a, stream);
        if (e != cudaSuccess) return e;
        a.least_rows = kFewRows + 1;
        a.most_rows = INT32_MAX;
    }
    return launch_kv_many(p, a, stream);
}

}  // namespace

size_t kv_attention_workspace_bytes(int head_dim, int group, int64_t max_new) {
    const size_t few = 2 * static_cast<size_t>(3 * sm_count()) * 16 * (head_dim + 2) * sizeof(float);
    return max_new * group <= kFewRows ? few : std::max(few, kv_many_workspace_bytes(head_dim));
}

cudaError_t launch_kv_attention(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
#define B200_KV_CASE(T, BITS, D) \
    if (p.bits == BITS && p.head_dim == D) return launch_attention<T, BITS, D>(p, a, stream);
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
