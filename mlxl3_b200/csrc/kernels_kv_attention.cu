// Attention of new tokens over a paged key/value cache: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the tokens j up to its own
// (with a window w: the last w of them).
//
// Work is shared out as kv_work.cuh says, in segments of 16 * WM rows and blocks of 64 keys.
//
// A block: 128 threads copy the keys and values (cp.async, 16 bytes each, several blocks in flight; what lies outside the
// visible range is filled with zeros, so nothing behind a length is ever multiplied), WK = 4 / WM warps take 64 / WK keys each
// against 16 rows: scores by mma.sync, online softmax in fp32 registers, probabilities rounded to 16 bits for the second product.
// Loads bound it: what a step of single tokens moves is the cache, once.
//
// Codes are multiplied as they are: 8- and 4-bit codes are exact in fp16, and so is what the tensor cores add up in fp32; the key's
// scale multiplies its scores, the value's its probability.  Those probabilities are taken relative to the largest value scale met so
// far (`unit`), so that rounding them to fp16 costs 2^-11 of what they weigh whatever the scales' magnitude.  bf16 queries enter fp16
// multiplied by a power of two of their own (exact but for what lies 2^-24 below the row's largest).
#include "kv_work.cuh"

#include <algorithm>

namespace b200exl3 {

namespace {

constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps;
constexpr int kFewKeys = 64;                       // keys of a block
constexpr int kFewCtasPerSm = 2;
constexpr int kFewTable = 128;
constexpr int kFewOver = 1;

template <int BITS, int D, int WM>
struct FewShape {
    static constexpr int kWk = kFewWarps / WM;     // warps that share the rows and take different keys
    static constexpr int kWarpKeys = kFewKeys / kWk;
    static constexpr int kRows = 16 * WM;
    static constexpr int kLanes = WM == 1 ? 1 : 32;    // a sequence has one row tile, or many
    static constexpr int kRowBytes = D * BITS / 8, kChunks = kRowBytes / 16;
    static constexpr int kTileBytes = kFewKeys * kRowBytes;
    static constexpr int kStageBytes = 2 * kTileBytes + (BITS == 16 ? 0 : 2 * kFewKeys * 4);
    static constexpr int kMergeStride = D + 4;
    static constexpr int kMergeBytes = kWk > 1 ? (kFewWarps / 2) * 16 * kMergeStride * 4 : 0;
    static constexpr bool kMergeInStage = kMergeBytes <= kStageBytes;      // the warps join in the block's own place where they fit
    static constexpr int kOwnMergeBytes = kMergeInStage ? 0 : kMergeBytes;
    static constexpr int kStages = std::min(6, (111 * 1024 - kOwnMergeBytes) / kStageBytes);      // two CTAs per SM
    static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + kOwnMergeBytes;
    static constexpr int kPartFloats = kRows * (D + 2);
};

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

// Where a 16-byte chunk of a tile's row lies: rows of 128 bytes and more swap their chunks by the row's number, shorter ones by the
// number of the 128 bytes they are in, so that eight rows' same chunk uses all banks.
template <int CHUNKS>
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
    constexpr int kShift = CHUNKS >= 8 ? 0 : (CHUNKS == 4 ? 1 : 2), kMask = CHUNKS >= 8 ? 7 : CHUNKS - 1;
    return static_cast<uint32_t>(row * CHUNKS + (chunk ^ ((row >> kShift) & kMask))) * 16;
}

// Two codes as fp16.  8 bits: bytes i and j of a word whose sign bits were flipped become 1024 + (code + 128); 4 bits: the low nibbles
// of its halves become 1024 + (code + 8).
__device__ __forceinline__ uint32_t less(uint32_t a, uint32_t bias) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&d);
}
template <int I, int J> __device__ __forceinline__ uint32_t codes8(uint32_t w) { return less(prmt(w, 0x64646464u, 0x4040u | I | (J << 8)), 0x64806480u); }
template <int I> __device__ __forceinline__ uint32_t codes4(uint32_t w) {
    uint32_t d;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(d) : "r"(w >> (4 * I)));    // (w & mask) | bias
    return less(d, 0x64086408u);
}

template <typename T, int BITS, int D, int WM>
__global__ void __launch_bounds__(kFewThreads, kFewCtasPerSm)
kv_few_kernel(const KvArgs p, const KvAttentionArgs a) {
    using S = FewShape<BITS, D, WM>;
    using M = std::conditional_t<BITS == 16, T, __half>;          // type of the products
    constexpr int kTiles = D / 8, kSteps = D / 16;                // column tiles of the output, steps of the first product
    constexpr int kNt = S::kWarpKeys / 8;                         // key tiles of a warp's block
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(128) unsigned char smem[];
    using Work = KvWork<S::kRows, kFewKeys, kFewOver>;
    using Cursor = KvCursor<S::kRows, kFewKeys, kFewOver>;
    __shared__ int64_t s_sum[kFewThreads / S::kLanes + 1];
    __shared__ KvTable<kFewTable> s_table;
    __shared__ Cursor s_cursor;
    __shared__ float2 s_ml[kFewWarps / 2][16];
    __shared__ bool s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int wm = warp % WM, wk = warp / WM;
    const Work work(p, a, s_table);
    KvRun run;
    if (!kv_find_run<kFewThreads, S::kLanes>(work, s_sum, s_cursor, run)) return;
    Cursor get = s_cursor;                                        // copies (put) run ahead of the products (get)
    if (get.block == get.end && !get.next_segment(work)) return;
    Cursor put = get;
    bool more = true;                                             // put stands at a block

    // ---- copies ------------------------------------------------------------------------------------------------------
    constexpr int kPerThread = kFewKeys * S::kChunks / kFewThreads, kRowStep = kFewThreads / S::kChunks;
    const int chunk = tid % S::kChunks, row0 = tid / S::kChunks;
    const uint32_t base = smem_addr(smem);
    int64_t place[kPerThread];                                    // of the next block to copy: its keys' vectors, or -1
    int64_t scale_place = -1;
    auto key_place = [&](int key) -> int64_t {
        return key >= put.seg.key0 && key < put.seg.key1 ? kv_place(p, put.b, key) : -1;
    };
    auto look_up = [&]() {
        const int first = put.seg.low + put.block * kFewKeys;
        const int64_t head = static_cast<int64_t>(put.head) * p.page_size;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            place[i] = key_place(first + row0 + i * kRowStep);
            if (place[i] >= 0) place[i] += head;
        }
        if constexpr (BITS != 16) {
            scale_place = key_place(first + (tid & 63));
            if (scale_place >= 0) scale_place += head;
        }
    };
    auto copy_block = [&](int stage) {
        const uint32_t dst = base + stage * S::kStageBytes;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const uint32_t at = dst + tile_at<S::kChunks>(row0 + i * kRowStep, chunk);
            const int64_t from = (place[i] < 0 ? 0 : place[i]) * S::kRowBytes + chunk * 16;
            copy16_fill(at, static_cast<const char*>(p.k) + from, place[i] >= 0);
            copy16_fill(at + S::kTileBytes, static_cast<const char*>(p.v) + from, place[i] >= 0);
        }
        if constexpr (BITS != 16)
            copy4_fill(dst + 2 * S::kTileBytes + tid * 4, (tid < kFewKeys ? p.k_scale : p.v_scale) + (scale_place < 0 ? 0 : scale_place), scale_place >= 0);
    };
    int asked = 0;
    auto ask = [&]() {
        if (more) {
            copy_block(asked);
            if (++asked == S::kStages) asked = 0;
            more = put.step(work);
            if (more) look_up();
        }
        copy_commit();
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) ask();

    // ---- state of a segment ---------------------------------------------------------------------------------------------
    uint32_t q[kSteps][4];
    float out[kTiles][4], m[2], l[2], unit = 0.0f, row_scale[2];
    int position[2];                                              // of this lane's two rows; -1: no row
    auto begin = [&]() {
        const int rows = work.rows_of(get.seq);
        const T* src[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = get.tile * S::kRows + wm * 16 + g + 8 * h;
            const int token = r / work.group;
            position[h] = r < rows ? get.seq.first_pos + token : -1;
            src[h] = r < rows ? static_cast<const T*>(a.q) + (get.seq.first_row + token) * a.q_stride +
                                    static_cast<int64_t>(get.head * work.group + r - token * work.group) * D
                              : nullptr;
            m[h] = -INFINITY;
            l[h] = 0.0f;
            row_scale[h] = a.scale_log2e;
        }
        unit = 0.0f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) out[i][0] = out[i][1] = out[i][2] = out[i][3] = 0.0f;
        // the order of the dimensions within a step is the one the keys come in
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int w = 0; w < 2; ++w)                           // columns 2t, 2t + 1 and 2t + 8, 2t + 9 of the step
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v = 0;
                    if (src[h] != nullptr) {
                        if constexpr (BITS == 16) v = *reinterpret_cast<const uint32_t*>(src[h] + s * 16 + 2 * t + 8 * w);
                        else if constexpr (BITS == 8) v = *reinterpret_cast<const uint32_t*>(src[h] + s * 16 + 4 * t + 2 * w);
                        else {
                            const uint16_t* e = reinterpret_cast<const uint16_t*>(src[h]) + (s >> 1) * 32 + 8 * t + 2 * (s & 1) + w;
                            v = e[0] | static_cast<uint32_t>(e[4]) << 16;
                        }
                    }
                    q[s][2 * w + h] = v;
                }
        if constexpr (!std::is_same_v<T, M>) {
            // bf16 rows enter fp16 products: scaled by the power of two that brings the row's largest to [1, 2)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float2 f = KvType<T>::unpack(q[s][2 * w + h]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
                // |e| <= 133: in two factors, each a normal number
                const float f0 = ldexpf(1.0f, -e / 2), f1 = ldexpf(1.0f, -e - -e / 2);
                row_scale[h] = ldexpf(row_scale[h], e);
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float2 f = KvType<T>::unpack(q[s][2 * w + h]);
                        q[s][2 * w + h] = KvType<M>::pack(f.x * f0 * f1, f.y * f0 * f1);
                    }
            }
        }
    };

    // ---- a block of a warp's keys ---------------------------------------------------------------------------------------
    auto multiply = [&](int stage) {
        const uint32_t keys = base + stage * S::kStageBytes, values = keys + S::kTileBytes;
        const int wrow = wk * S::kWarpKeys;
        const int mrow = (lane & 7) + ((lane >> 4) << 3), mchunk = (lane >> 3) & 1;     // matrices of keys: (octet, chunk) = (0, 0) (0, 1) (1, 0) (1, 1)
        float s[kNt][4];
#pragma unroll
        for (int i = 0; i < kNt; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::kChunks; c += 2)
#pragma unroll
            for (int i = 0; i < kNt; i += 2) {
                uint32_t r[4];
                ldmatrix4(keys + tile_at<S::kChunks>(wrow + i * 8 + mrow, c + mchunk), r);
                if constexpr (BITS == 16) {
                    mma_rows<M>(s[i], q[c / 2], r[0], r[1]);
                    mma_rows<M>(s[i + 1], q[c / 2], r[2], r[3]);
                } else if constexpr (BITS == 8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t w = r[j] ^ 0x80808080u;
                        mma_rows<M>(s[i + (j >> 1)], q[c + (j & 1)], codes8<0, 1>(w), codes8<2, 3>(w));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_rows<M>(s[i + (j >> 1)], q[2 * (c + (j & 1))], codes4<0>(r[j]), codes4<1>(r[j]));
                        mma_rows<M>(s[i + (j >> 1)], q[2 * (c + (j & 1)) + 1], codes4<2>(r[j]), codes4<3>(r[j]));
                    }
                }
            }
        const float* scales = reinterpret_cast<const float*>(smem + stage * S::kStageBytes + 2 * S::kTileBytes) + wrow + 2 * t;
        float2 vs[kNt];
        float unit_ratio = 1.0f;
        if constexpr (BITS != 16) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kNt; ++i) {
                const float2 ks = *reinterpret_cast<const float2*>(scales + i * 8);
                vs[i] = *reinterpret_cast<const float2*>(scales + kFewKeys + i * 8);
                top = fmaxf(top, fmaxf(vs[i].x, vs[i].y));
                s[i][0] *= ks.x; s[i][1] *= ks.y; s[i][2] *= ks.x; s[i][3] *= ks.y;
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (top > unit) {
                unit_ratio = unit / top;
                unit = top;
            }
            const float inverse = unit > 0.0f ? 1.0f / unit : 0.0f;
#pragma unroll
            for (int i = 0; i < kNt; ++i) { vs[i].x *= inverse; vs[i].y *= inverse; }
        }
        // masks, maximum, probabilities
        const int first = get.seg.low + get.block * kFewKeys + wrow + 2 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int end = min(position[h] + 1, work.capacity);
            const int start = a.window > 0 ? position[h] + 1 - a.window : 0;
            float top = m[h];
#pragma unroll
            for (int i = 0; i < kNt; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = first + i * 8 + e;
                    float& x = s[i][2 * h + e];
                    x = key < end && key >= start ? x * row_scale[h] : -INFINITY;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float safe = top == -INFINITY ? 0.0f : top;     // a row that saw nothing yet
            const float correction = exp2_fast(m[h] - safe);
            m[h] = top;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kNt; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = s[i][2 * h + e];
                    x = exp2_fast(x - safe);
                    sum += x;
                    if constexpr (BITS != 16) x *= e ? vs[i].y : vs[i].x;
                }
            l[h] = fmaf(l[h], correction, sum);
            const float factor = BITS == 16 ? correction : correction * unit_ratio;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) { out[i][2 * h] *= factor; out[i][2 * h + 1] *= factor; }
        }
        // probabilities times values
        const int vrow = (lane & 7) + ((lane >> 3) & 1) * 8, vchunk = lane >> 4;         // matrices of values: (octet, chunk) = (0, 0) (1, 0) (0, 1) (1, 1)
#pragma unroll
        for (int k = 0; k < kNt / 2; ++k) {
            const uint32_t pr[4] = {KvType<M>::pack(s[2 * k][0], s[2 * k][1]), KvType<M>::pack(s[2 * k][2], s[2 * k][3]),
                                    KvType<M>::pack(s[2 * k + 1][0], s[2 * k + 1][1]), KvType<M>::pack(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
            for (int c = 0; c < S::kChunks; c += 2) {
                uint32_t r[4];
                ldmatrix4_trans(values + tile_at<S::kChunks>(wrow + k * 16 + vrow, c + vchunk), r);
                if constexpr (BITS == 16) {
                    mma_rows<M>(out[c], pr, r[0], r[1]);
                    mma_rows<M>(out[c + 1], pr, r[2], r[3]);
                } else if constexpr (BITS == 8) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t w0 = r[2 * j] ^ 0x80808080u, w1 = r[2 * j + 1] ^ 0x80808080u;
                        mma_rows<M>(out[2 * (c + j)], pr, codes8<0, 2>(w0), codes8<0, 2>(w1));
                        mma_rows<M>(out[2 * (c + j) + 1], pr, codes8<1, 3>(w0), codes8<1, 3>(w1));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_rows<M>(out[4 * (c + j)], pr, codes4<0>(r[2 * j]), codes4<0>(r[2 * j + 1]));
                        mma_rows<M>(out[4 * (c + j) + 1], pr, codes4<1>(r[2 * j]), codes4<1>(r[2 * j + 1]));
                        mma_rows<M>(out[4 * (c + j) + 2], pr, codes4<2>(r[2 * j]), codes4<2>(r[2 * j + 1]));
                        mma_rows<M>(out[4 * (c + j) + 3], pr, codes4<3>(r[2 * j]), codes4<3>(r[2 * j + 1]));
                    }
                }
            }
        }
    };
    // dimension of out[i][e] (e = 0, 1): where the values' chunks put it
    auto dim_of = [&](int i, int e) {
        if constexpr (BITS == 16) return i * 8 + 2 * t + e;
        else if constexpr (BITS == 8) return (i >> 1) * 16 + 2 * (2 * t + e) + (i & 1);
        else return (i >> 2) * 32 + 4 * (2 * t + e) + (i & 3);
    };

    // ---- end of a segment, or of this CTA's part of it ----------------------------------------------------------------
    auto store_row = [&](int r, int d, float v0, float v1, bool pair) {     // row r of the segment's sequence
        const int token = r / work.group;
        T* dst = static_cast<T*>(a.out) + (get.seq.first_row + token) * a.out_stride + static_cast<int64_t>(get.head * work.group + r - token * work.group) * D + d;
        const uint32_t w = KvType<T>::pack(v0, v1);
        if (pair) *reinterpret_cast<uint32_t*>(dst) = w;
        else *dst = reinterpret_cast<const T*>(&w)[0];
    };
    auto finish = [&](int stage) {
        float* merge = reinterpret_cast<float*>(smem + (S::kMergeInStage ? stage : S::kStages) * S::kStageBytes);
        if constexpr (S::kMergeInStage && S::kWk > 1) __syncthreads();     // every warp is through with the block
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        if constexpr (BITS != 16) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) out[i][e] *= unit;
        }
        // the warps that took other keys of the same rows, the upper half into the lower
#pragma unroll
        for (int half = S::kWk / 2; half >= 1; half >>= 1) {
            if (wk >= half && wk < 2 * half) {
                float* dst = merge + ((wk - half) * WM + wm) * 16 * S::kMergeStride;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (t == 0) s_ml[(wk - half) * WM + wm][g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e) dst[(g + 8 * h) * S::kMergeStride + i * 8 + 2 * t + e] = out[i][2 * h + e];
                }
            }
            __syncthreads();
            if (wk < half) {
                const float* src = merge + (wk * WM + wm) * 16 * S::kMergeStride;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 o = s_ml[wk * WM + wm][g + 8 * h];
                    const float top = fmaxf(m[h], o.x), safe = top == -INFINITY ? 0.0f : top;
                    const float c0 = exp2_fast(m[h] - safe), c1 = exp2_fast(o.x - safe);
                    m[h] = top;
                    l[h] = l[h] * c0 + o.y * c1;
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            out[i][2 * h + e] = out[i][2 * h + e] * c0 + src[(g + 8 * h) * S::kMergeStride + i * 8 + 2 * t + e] * c1;
                }
            }
            __syncthreads();
        }
        const int rows = work.rows_of(get.seq), tile0 = get.tile * S::kRows;
        const int64_t first_unit = get.base + kFewOver;
        const int c0 = run.cta_of(first_unit), c1 = run.cta_of(first_unit + get.seg.blocks - 1);     // CTAs that hold its first and last block
        if (c0 == c1) {
            if (wk == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = tile0 + wm * 16 + g + 8 * h;
                    if (r >= rows) continue;
                    const float inverse = kv_inverse(l[h]);
#pragma unroll
                    for (int i = 0; i < kTiles; ++i) {
                        if constexpr (BITS == 16) {
                            store_row(r, dim_of(i, 0), out[i][2 * h] * inverse, out[i][2 * h + 1] * inverse, true);
                        } else {
                            store_row(r, dim_of(i, 0), out[i][2 * h] * inverse, 0.0f, false);
                            store_row(r, dim_of(i, 1), out[i][2 * h + 1] * inverse, 0.0f, false);
                        }
                    }
                }
            }
            return;
        }
        // this CTA's part: its first place for a segment that began before its run, else the second
        auto part_of = [&](int c) { return a.parts + (2 * c + (c == c0 ? 1 : 0)) * static_cast<int64_t>(S::kPartFloats); };
        float* part = part_of(blockIdx.x);
        if (wk == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = wm * 16 + g + 8 * h;
                if (tile0 + r >= rows) continue;
                if (t == 0) reinterpret_cast<float2*>(part + S::kRows * D)[r] = make_float2(m[h], l[h]);
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) part[r * D + dim_of(i, e)] = out[i][2 * h + e];
            }
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const unsigned int before = atomicAdd(a.arrived + c0, 1u);
            s_last = before == static_cast<unsigned int>(c1 - c0);
            if (s_last) a.arrived[c0] = 0;                        // the next call starts from zero
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        // a warp joins a row: its lanes weigh the parts, then every lane adds its dimensions over the parts in order
        const int parts = c1 - c0 + 1, rows_here = min(S::kRows, rows - tile0);
        for (int r = warp; r < rows_here; r += kFewWarps) {
            auto weight_of = [&](int q_) { return __ldcg(reinterpret_cast<const float2*>(part_of(c0 + q_) + S::kRows * D) + r); };
            float top = -INFINITY;
            for (int q_ = lane; q_ < parts; q_ += 32) top = fmaxf(top, weight_of(q_).x);
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float safe = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, o[D / 32];
#pragma unroll
            for (int e = 0; e < D / 32; ++e) o[e] = 0.0f;
            for (int q0 = 0; q0 < parts; q0 += 32) {
                float2 ml = make_float2(-INFINITY, 0.0f);
                if (q0 + lane < parts) ml = weight_of(q0 + lane);
                const float c = exp2_fast(ml.x - safe);
                sum += c * ml.y;
                const int n = min(32, parts - q0);
#pragma unroll 8
                for (int i = 0; i < n; ++i) {
                    const float w = __shfl_sync(0xffffffffu, c, i);
                    const float* src = part_of(c0 + q0 + i) + r * D;
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) o[e] = fmaf(__ldcg(src + lane * (D / 32) + e), w, o[e]);
                }
            }
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const float inverse = kv_inverse(sum);
#pragma unroll
            for (int e = 0; e < D / 32; e += 2) store_row(tile0 + r, lane * (D / 32) + e, o[e] * inverse, o[e + 1] * inverse, true);
        }
    };

    // ---- the run ------------------------------------------------------------------------------------------------------
    begin();
    for (int stage = 0;; stage = stage + 1 == S::kStages ? 0 : stage + 1) {
        copy_wait<S::kStages - 2>();
        __syncthreads();                                          // the block has landed, and the one before was used by all
        ask();
        multiply(stage);
        if (++get.block == get.end) {
            finish(stage);
            if (!get.next_segment(work)) break;
            begin();
        }
    }
}

template <typename T, int BITS, int D, int WM>
cudaError_t launch_few(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
    using S = FewShape<BITS, D, WM>;
    static PerDeviceOnce attribute;
    if (attribute.needed()) {
        cudaError_t e = cudaFuncSetAttribute(kv_few_kernel<T, BITS, D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        attribute.mark();
    }
    return launch_dependent(kv_few_kernel<T, BITS, D, WM>, dim3(static_cast<unsigned>(kFewCtasPerSm * sm_count())), dim3(kFewThreads), S::kSmem, stream, p, a);
}

// Up to this many rows per key head the few-row kernel takes a sequence.
constexpr int kFewRows = 16;

template <typename T, int BITS, int D>
cudaError_t launch_attention(const KvArgs& p, KvAttentionArgs a, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.max_new) * (a.heads / p.kv_heads);
    a.least_rows = 1;
    a.most_rows = INT32_MAX;
    if (rows <= kFewRows) return launch_few<T, BITS, D, 1>(p, a, stream);
    if constexpr (BITS != 16) {
        return launch_few<T, BITS, D, 4>(p, a, stream);
    } else {
        if (p.batch > 1) {                                        // sequences of few rows among the others
            a.most_rows = kFewRows;
            const cudaError_t e = launch_few<T, BITS, D, 1>(p, a, stream);
            if (e != cudaSuccess) return e;
            a.least_rows = kFewRows + 1;
            a.most_rows = INT32_MAX;
        }
        return launch_kv_many(p, a, stream);
    }
}

}  // namespace

size_t kv_attention_workspace_bytes(int bits, int head_dim, int group, int64_t max_new) {
    const size_t few = 2 * static_cast<size_t>(kFewCtasPerSm * sm_count()) * (bits == 16 ? 16 : 64) * (head_dim + 2) * sizeof(float);
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
