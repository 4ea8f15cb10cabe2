// Attention of many new tokens over a paged key/value cache (prompts, chunks of prompts, draft tokens of wide groups) on the tcgen05
// tensor cores; kernels_kv_attention.cu has the mathematics and takes the sequences of few rows.
//
// A segment is 256 rows of a sequence and key head, its keys come in blocks of 128 (kv_work.cuh).  Per block, tile x (128 rows) of
// the segment: S_x = Q_x K^T (128 x 128, fp32, tensor memory), probabilities P_x = exp2(S_x scale - m) by the 128 threads that own one
// row each, rounded to 16 bits and stored over the half of S_x that was read first, then O_x += P_x V with P_x as the tensor-memory
// operand.  The two tiles share the block's keys and values and take turns: while the tensor cores multiply for one, the other's
// exponentials are computed.  Tensor memory: S_0, S_1, O_0, O_1.
//
// The running maximum m of a row is moved only when a score exceeds it by 2^8 (in log2 units 8): until then probabilities may reach
// 256, which 16 bits hold as well as 1, and O_x and the sum stay in the same unit.  When it moves, the row's thread rescales O_x in
// tensor memory; S_x of a block being complete implies that the product before it is, so nothing else has to be waited for.
//
// Four warps bring the data: cp.async, 16 bytes each, zeros for what lies outside the visible range, into the 128-byte swizzle that the
// products read.  One thread issues the products.  Every wait is bounded; one that gives up sets the status word, all roles run on
// to the end, and the kernel frees its tensor memory.
#include "kv_work.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <type_traits>

namespace b200exl3 {

namespace {

constexpr int kManyKeys = 128, kManyTile = 128, kManyRows = 2 * kManyTile;
constexpr int kSoftmaxWarps = 8, kLoadWarps = 4;
constexpr int kLoadThreads = 32 * kLoadWarps;
constexpr int kManyThreads = 32 * (kSoftmaxWarps + kLoadWarps + 1);
constexpr int kManyTable = 512;
constexpr uint32_t kScoreCols = 128;               // tensor-memory columns of S_x; P_x lies in their second half

template <int BITS, int D>
struct ManyShape {
    static constexpr int kTileBytes = kManyKeys * D * 2;           // a block's keys or values, as the products read them
    static constexpr int kSlots = D == 128 ? 4 : 6;                // keys and values in flight, alternately
    static constexpr int kQueryBytes = kManyRows * D * 2;
    static constexpr size_t kSmem = 1024 + kQueryBytes + static_cast<size_t>(kSlots) * kTileBytes;
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

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kManyThreads, 1)
kv_many_kernel(const KvArgs p, const KvAttentionArgs a) {
    using S = ManyShape<BITS, D>;
    using Work = KvWork<kManyRows, kManyKeys>;
    using Cursor = KvCursor<kManyRows, kManyKeys>;
    constexpr int kChunks = D / 8;
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ KvTable<kManyTable> s_table;
    __shared__ int64_t s_sum[kManyThreads / 32 + 1];
    __shared__ Cursor s_cursor;
    __shared__ __align__(8) uint64_t kv_full[S::kSlots], kv_free[S::kSlots], s_full[2], p_full[2], o_full[2], q_free, drained;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int s_last[2];
    __shared__ volatile int s_failed;

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const Work work(p, a, s_table);
    KvRun run;
    if (!kv_find_run<kManyThreads, 32>(work, s_sum, s_cursor, run)) return;
    const int count = static_cast<int>(run.u1 - run.u0);
    unsigned char* const queries = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    unsigned char* const tiles = queries + S::kQueryBytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kSlots; ++s) { mbar_init(&kv_full[s], kLoadThreads); mbar_init(&kv_free[s], 1); }
        for (int x = 0; x < 2; ++x) { mbar_init(&s_full[x], 1); mbar_init(&p_full[x], kManyTile); mbar_init(&o_full[x], 1); }
        mbar_init(&q_free, 1);
        mbar_init(&drained, 1);
        s_failed = 0;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == kSoftmaxWarps + kLoadWarps) tmem_alloc(&tmem_base_slot, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base_slot;

    if (warp < kSoftmaxWarps) {
        // ================= rows: one thread each =================
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t scores = tmem + lanes + x * kScoreCols, probs = scores + kScoreCols / 2, outs = tmem + lanes + S::kOutCols + x * D;
        Cursor at = s_cursor;
        uint32_t s_par = 0, o_par = 0;
        int done = 0;
        int64_t seg_begin = run.u0 - at.block;
        while (done < count) {
            const int rows = work.rows_of(at.seq), row = at.tile * kManyRows + x * kManyTile + r;
            const int n = min(count - done, at.seg.blocks - at.block);
            const bool two = rows - at.tile * kManyRows > kManyTile;
            if (x == 0 || two) {
                const int token = row / work.group;
                const bool live = row < rows;
                const int position = live ? at.seq.first_pos + token : -1;
                const int end = min(position + 1, work.capacity), start = a.window > 0 ? position + 1 - a.window : 0;
                float m = -INFINITY, l = 0.0f;
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    const int first = at.seg.low + (at.block + j) * kManyKeys;
                    const int e = end - first, b = start - first;              // visible: columns b .. e - 1
                    qmm_wait(&s_full[x], s_par, &s_failed);
                    s_par ^= 1u;
                    __syncwarp();
                    fence_after();
                    const bool masked = __any_sync(0xffffffffu, e < kManyKeys || b > 0);
                    uint32_t v0[32], v1[32];
                    auto largest = [&](uint32_t (&v)[32], int col, float top) {
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = col + i < e && col + i >= b ? v[i] : 0xff800000u;
                        }
                        float t0 = top, t1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            t0 = fmaxf(t0, __uint_as_float(v[i]));
                            t1 = fmaxf(t1, __uint_as_float(v[i + 1]));
                        }
                        return fmaxf(t0, t1);
                    };
                    float top = -INFINITY;
                    tmem_ld32(scores, v0);
                    tmem_ld32(scores + 32, v1);
                    tmem_wait_ld();
                    top = largest(v0, 0, top);
                    top = largest(v1, 32, top);
                    __syncwarp();
                    tmem_ld32(scores + 64, v0);
                    tmem_ld32(scores + 96, v1);
                    tmem_wait_ld();
                    top = largest(v0, 64, top);
                    top = largest(v1, 96, top);
                    top *= a.scale_log2e;
                    const bool moves = top > m + 8.0f;                           // also from -inf
                    if (__any_sync(0xffffffffu, moves)) {
                        const float to = moves ? top : m;
                        const float factor = moves ? exp2_fast(m - to) : 1.0f;
                        m = to;
                        l *= factor;
                        if (j > 0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                __syncwarp();
                                asm volatile(
                                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                                    : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
                                      "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                                    : "r"(outs + c) : "memory");
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                                tmem_st16(outs + c, o);
                            }
                        }
                    }
                    const float shift = m == -INFINITY ? 0.0f : -m;
                    // columns 64 .. 127 are in registers; their probabilities go where those scores lay, then columns 0 .. 63
                    float l0 = 0.0f, l1 = 0.0f;
                    auto put = [&](uint32_t (&v)[32], int col) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float p0 = exp2_fast(fmaf(__uint_as_float(v[2 * i]), a.scale_log2e, shift));
                            const float p1 = exp2_fast(fmaf(__uint_as_float(v[2 * i + 1]), a.scale_log2e, shift));
                            l0 += p0;
                            l1 += p1;
                            w[i] = KvType<T>::pack(p0, p1);
                        }
                        __syncwarp();
                        tmem_st16(probs + col / 2, w);
                    };
                    put(v0, 64);
                    put(v1, 96);
                    tmem_ld32(scores, v0);
                    tmem_ld32(scores + 32, v1);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            v0[i] = i < e && i >= b ? v0[i] : 0xff800000u;
                            v1[i] = 32 + i < e && 32 + i >= b ? v1[i] : 0xff800000u;
                        }
                    }
                    put(v0, 0);
                    put(v1, 32);
                    l += l0 + l1;
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(&p_full[x]);
                }
                // ---- the segment's rows, or this CTA's part of them
                qmm_wait(&o_full[x], o_par, &s_failed);
                o_par ^= 1u;
                __syncwarp();
                fence_after();
                const int c0 = run.cta_of(seg_begin), c1 = run.cta_of(seg_begin + at.seg.blocks - 1);
                T* const dst = static_cast<T*>(a.out) + (at.seq.first_row + token) * a.out_stride +
                               static_cast<int64_t>(at.head * work.group + row - token * work.group) * D;
                auto part_of = [&](int c) { return a.parts + (2 * c + (c == c0 ? 1 : 0)) * static_cast<int64_t>(S::kPartFloats); };
                const int pr = x * kManyTile + r;
                const bool whole = c0 == c1;
                const float inverse = kv_inverse(l);
                float* const mine = whole ? nullptr : part_of(blockIdx.x) + pr * D;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(outs + c, v);
                    tmem_wait_ld();
                    if (!live) continue;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                w[k] = KvType<T>::pack(__uint_as_float(v[i + 2 * k]) * inverse, __uint_as_float(v[i + 2 * k + 1]) * inverse);
                            *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(mine + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                }
                fence_before();
                if (!whole) {
                    if (live) reinterpret_cast<float2*>(part_of(blockIdx.x) + kManyRows * D)[pr] = make_float2(m, l);
                    __threadfence();
                    group_sync(1 + x, kManyTile);
                    if (r == 0) {
                        unsigned int* counter = a.arrived + 2 * c0 + x;
                        s_last[x] = atomicAdd(counter, 1u) == static_cast<unsigned int>(c1 - c0);
                        if (s_last[x]) *counter = 0;                              // the next call starts from zero
                    }
                    group_sync(1 + x, kManyTile);
                    if (s_last[x] && live) {
                        __threadfence();
                        auto weight_of = [&](int c) { return __ldcg(reinterpret_cast<const float2*>(part_of(c) + kManyRows * D) + pr); };
                        float top = -INFINITY, sum = 0.0f;
                        for (int c = c0; c <= c1; ++c) top = fmaxf(top, weight_of(c).x);
                        const float safe = top == -INFINITY ? 0.0f : top;
                        for (int c = c0; c <= c1; ++c) {
                            const float2 ml = weight_of(c);
                            sum = fmaf(exp2_fast(ml.x - safe), ml.y, sum);
                        }
                        const float inv = kv_inverse(sum);
#pragma unroll 1
                        for (int d = 0; d < D; d += 32) {
                            float4 o[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            for (int c = c0; c <= c1; ++c) {
                                const float w = exp2_fast(weight_of(c).x - safe);
                                const float4* src = reinterpret_cast<const float4*>(part_of(c) + pr * D + d);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float4 f = __ldcg(src + i);
                                    o[i].x = fmaf(f.x, w, o[i].x); o[i].y = fmaf(f.y, w, o[i].y); o[i].z = fmaf(f.z, w, o[i].z); o[i].w = fmaf(f.w, w, o[i].w);
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 8; i += 2)
                                *reinterpret_cast<uint4*>(dst + d + 4 * i) =
                                    make_uint4(KvType<T>::pack(o[i].x * inv, o[i].y * inv), KvType<T>::pack(o[i].z * inv, o[i].w * inv),
                                               KvType<T>::pack(o[i + 1].x * inv, o[i + 1].y * inv), KvType<T>::pack(o[i + 1].z * inv, o[i + 1].w * inv));
                        }
                    }
                    __syncwarp();
                }
            }
            done += n;
            seg_begin += at.seg.blocks;
            if (done < count) at.next_segment(work);
        }
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        // ================= copies =================
        const int tid = threadIdx.x - 32 * kSoftmaxWarps;
        constexpr int kRowStep = kLoadThreads / kChunks, kPer = kManyKeys / kRowStep;
        const int chunk = tid % kChunks, row0 = tid / kChunks;
        const uint32_t q_base = smem_addr(queries), tile_base = smem_addr(tiles);
        Cursor at = s_cursor;
        int issued = 0, told = 0;                                 // tiles asked for; tiles whose arrival was announced
        auto announce = [&](int upto) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (; told < upto; ++told) mbar_arrive(&kv_full[told % S::kSlots]);
        };
        uint32_t segments = 0;
        int done = 0;
        while (done < count) {
            const int rows = work.rows_of(at.seq), tile0 = at.tile * kManyRows;
            const int n = min(count - done, at.seg.blocks - at.block);
            if (segments > 0) {
                copy_wait<0>();
                announce(issued);                                 // the products that free the queries wait for these
                qmm_wait(&q_free, (segments - 1) & 1u, &s_failed);
                __syncwarp();
            }
            ++segments;
            // queries of both tiles; rows past the last are zeros
#pragma unroll 4
            for (int r = row0; r < kManyRows; r += kRowStep) {
                const int row = tile0 + r, token = row / work.group;
                const bool live = row < rows;
                const T* src = static_cast<const T*>(a.q) + (live ? (at.seq.first_row + token) * a.q_stride +
                                                                       static_cast<int64_t>(at.head * work.group + row - token * work.group) * D + chunk * 8
                                                                  : 0);
                copy16_fill(q_base + (r >> 7) * (S::kQueryBytes / 2) + many_at(kManyTile, r & 127, chunk), src, live);
            }
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                const int first = at.seg.low + (at.block + j) * kManyKeys;
                int64_t place[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int key = first + row0 + i * kRowStep;
                    place[i] = key >= at.seg.key0 && key < at.seg.key1 ? kv_place(p, at.b, key) : -1;
                    if (place[i] >= 0) place[i] += static_cast<int64_t>(at.head) * p.page_size;
                }
#pragma unroll
                for (int kind = 0; kind < 2; ++kind) {            // keys, values
                    const int slot = issued % S::kSlots;
                    if (issued >= S::kSlots) {
                        qmm_wait(&kv_free[slot], (issued / S::kSlots - 1) & 1u, &s_failed);
                        __syncwarp();
                    }
                    const char* pool = static_cast<const char*>(kind ? p.v : p.k) + chunk * 16;
                    const uint32_t dst = tile_base + slot * S::kTileBytes;
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        copy16_fill(dst + many_at(kManyKeys, row0 + i * kRowStep, chunk), pool + (place[i] < 0 ? 0 : place[i] * (D * 2)), place[i] >= 0);
                    copy_commit();
                    ++issued;
                    copy_wait<2>();
                    announce(issued - 2);
                }
            }
            done += n;
            if (done < count) at.next_segment(work);
        }
        copy_wait<0>();
        announce(issued);
    } else if (elect_one()) {
        // ================= products =================
        constexpr uint32_t kFormat = std::is_same_v<T, __half> ? 0u : 1u;
        constexpr uint32_t kBase = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((128u >> 4) << 24);
        constexpr uint32_t kScoreDesc = kBase | ((static_cast<uint32_t>(kManyKeys) >> 3) << 17);
        constexpr uint32_t kValueDesc = kBase | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17);    // values: N is the contiguous axis
        const uint64_t q_desc = umma_desc(smem_addr(queries)), k_desc = umma_desc(smem_addr(tiles));
        const uint64_t v_desc = umma_desc_values(smem_addr(tiles), kManyKeys * 128);
        Cursor at = s_cursor;
        int tile = 0, done = 0;                                   // tiles consumed
        uint32_t p_par[2] = {0, 0};
        auto wait_tile = [&](int i) {
            qmm_wait(&kv_full[i % S::kSlots], (i / S::kSlots) & 1u, &s_failed);
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
        };
        auto weigh = [&](int x, int slot, bool accumulate) {
            qmm_wait(&p_full[x], p_par[x], &s_failed);
            p_par[x] ^= 1u;
            fence_after();
            const uint64_t vd = v_desc + slot * (S::kTileBytes >> 4);
#pragma unroll
            for (int k = 0; k < kManyKeys / 16; ++k)
                umma_f16_ts(tmem + S::kOutCols + x * D, tmem + x * kScoreCols + kScoreCols / 2 + k * 8, vd + k * (16 * 128 >> 4), kValueDesc,
                            accumulate || k > 0);
        };
        while (done < count) {
            const int rows = work.rows_of(at.seq);
            const int n = min(count - done, at.seg.blocks - at.block);
            const bool two = rows - at.tile * kManyRows > kManyTile;
            wait_tile(tile);
            score(0, tile % S::kSlots);
            if (two) score(1, tile % S::kSlots);
            umma_commit(&kv_free[tile % S::kSlots]);
            if (n == 1) umma_commit(&q_free);
            for (int j = 0; j < n; ++j) {
                const int vt = tile + 1, kt = tile + 2;
                const bool more = j + 1 < n;
                wait_tile(vt);
                weigh(0, vt % S::kSlots, j > 0);
                if (more) {
                    wait_tile(kt);
                    score(0, kt % S::kSlots);
                } else {
                    umma_commit(&o_full[0]);
                }
                if (two) {
                    weigh(1, vt % S::kSlots, j > 0);
                    umma_commit(&kv_free[vt % S::kSlots]);
                    if (more) score(1, kt % S::kSlots);
                    else umma_commit(&o_full[1]);
                } else {
                    umma_commit(&kv_free[vt % S::kSlots]);
                }
                if (more) {
                    umma_commit(&kv_free[kt % S::kSlots]);
                    if (j + 2 == n) umma_commit(&q_free);
                }
                tile += 2;
            }
            done += n;
            if (done < count) at.next_segment(work);
        }
        umma_commit(&drained);
        qmm_wait(&drained, 0, &s_failed);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kSoftmaxWarps + kLoadWarps) {
        __syncwarp();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && s_failed) atomicExch(a.error, 8u);
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
    return launch_dependent(kv_many_kernel<T, BITS, D>, dim3(static_cast<unsigned>(sm_count())), dim3(kManyThreads), S::kSmem, stream, p, a);
}

}  // namespace

size_t kv_many_workspace_bytes(int head_dim) { return 2 * static_cast<size_t>(sm_count()) * kManyRows * (head_dim + 2) * sizeof(float); }

cudaError_t launch_kv_many(const KvArgs& p, const KvAttentionArgs& a, cudaStream_t stream) {
    if (p.dtype == kF16) return p.head_dim == 128 ? launch_many<__half, 16, 128>(p, a, stream) : launch_many<__half, 16, 64>(p, a, stream);
    return p.head_dim == 128 ? launch_many<__nv_bfloat16, 16, 128>(p, a, stream) : launch_many<__nv_bfloat16, 16, 64>(p, a, stream);
}

}  // namespace b200exl3
