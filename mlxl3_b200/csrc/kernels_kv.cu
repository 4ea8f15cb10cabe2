// Rotary embedding with the append to a paged key/value cache, and reading the cache back.
//
// append: row i of a sequence's n new rows is its token at position p = length - n + i.  The pairs (a, b) of the first `rotated`
// dimensions of every q and k head -- (j, j + rotated/2), or (2j, 2j + 1) interleaved -- turn by the angle 2 pi p f_j, f_j in turns
// per position: (a, b) -> m (a cos - b sin, a sin + b cos).  The product p f_j is taken in 64 bits and only its fraction goes into
// sine and cosine, so a token at position 10^6 is as exact as the first; both are computed in 64 bits once per token and pair and
// shared by all heads.  q goes to a buffer of its own (or in place), k and v to row p % page_size of the sequence's page
// p / page_size.
//
// A quantised cache holds a vector x as codes round(x m / max|x|), m = 127 or 7, and one fp32 scale max|x| / m.  The rotated k is kept
// in 64 bits up to the code: between two codes a last bit of fp32 decides, and every element of a long cache gets its chance at it.
// v needs no more than fp32: x m is exact there (from 2^100 on after a step by a power of two) and the quotient of two 16-bit values is
// never closer to a border than that division rounds, unless it lies on it.  4-bit codes are stored as code + 8, the even dimension in the
// low half of the byte.
//
// Both kernels are bound by memory (and short calls by the chain row_start -> length -> page table -> data): 16 or 8 lanes hold a
// vector, 8 dimensions each, so that every access is 16 bytes (8 or 4 for codes) and a vector one coalesced piece.  Three prompts of 6674
// rows, 32 heads over 8 of 128, fp16: 37 us, 68 % of the measured copy rate; with the angles read from shared memory for every vector
// and four rows one after the other 83 us.  4000 rows into 4 bits: 50 us, bound by the instructions of the 64-bit path (four CTAs per
// SM; three 63 with the reading back where four take 58).  60001 rows out of 4 bits: 61.5 us, 77 %.
#include <algorithm>
#include <type_traits>

#include "kv_work.cuh"

namespace b200exl3 {

namespace {

constexpr int kKvThreads = 256;
constexpr int kKvStarts = 256;              // sequences whose first rows are searched in shared memory

// Sequence of a row: the last one that starts at or before it, by bisection (rows ascend from sequence to sequence).
template <typename Start>
__device__ __forceinline__ int kv_find(int batch, int row, Start start) {
    int low = 0, high = batch;              // start(low) <= row, or low == 0
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (start(mid) <= row) low = mid; else high = mid;
    }
    return low;
}

struct KvRow {
    int64_t place;          // vector of head 0, or -1: not in the cache
    int pos;                // position, or -1: no sequence's row
};

// Where the ROWS rows from row0 on belong: one thread per row, after the first rows were brought to shared memory.
template <int ROWS>
__device__ __forceinline__ void kv_locate(const KvArgs& p, int64_t row0, int (&s_start)[kKvStarts + 1], KvRow (&s_row)[ROWS]) {
    const bool shared = p.batch <= kKvStarts;
    if (shared) {
        for (int i = threadIdx.x; i <= p.batch; i += kKvThreads) s_start[i] = kv_clamp_row(p, __ldg(p.row_start + i));
        __syncthreads();
    }
    if (threadIdx.x < ROWS) {
        KvRow r{-1, -1};
        if (row0 + threadIdx.x < p.rows) {
            const int row = static_cast<int>(row0) + static_cast<int>(threadIdx.x);
            auto start = [&](int b) { return shared ? s_start[b] : kv_clamp_row(p, __ldg(p.row_start + b)); };
            int b = kv_find(p.batch, row, start);
            const int first = start(b), end = start(b + 1);
            if (row >= first && row < end) {
                const int pos = kv_clamp_length(__ldg(p.length + b)) - end + row;
                if (pos >= 0) {
                    r.pos = pos;
                    r.place = kv_place(p, b, pos);
                }
            }
        }
        s_row[threadIdx.x] = r;
    }
    __syncthreads();
}

__device__ __forceinline__ double kv_abs_max(double m, double x) { x = fabs(x); return x > m || x != x ? x : m; }
__device__ __forceinline__ float kv_abs_max(float m, float x) { x = fabsf(x); return x > m || x != x ? x : m; }
__device__ __forceinline__ double kv_divide(double a, double b) { return __ddiv_rn(a, b); }
__device__ __forceinline__ float kv_divide(float a, float b) { return __fdiv_rn(a, b); }
// The whole number nearest to t, |t| < 2^20, and t's distance from it
__device__ __forceinline__ int kv_nearest(double t, double& off) {
    const double r = __dadd_rn(t, 6755399441055744.0);            // 1.5 * 2^52
    off = t - __dsub_rn(r, 6755399441055744.0);
    return __double2loint(r);
}
__device__ __forceinline__ int kv_nearest(float t, float& off) {
    const float r = __fadd_rn(t, 12582912.0f);                    // 1.5 * 2^23
    off = t - __fsub_rn(r, 12582912.0f);
    return static_cast<int>(__float_as_uint(r) << 10) >> 10;
}

// Codes of eight dimensions of a vector that LANES neighbouring lanes hold, and its scale.  A NaN or an infinity anywhere is the
// scale, with codes of 0: the whole vector reads as NaN.
template <int BITS, int LANES, typename F>
__device__ __forceinline__ void kv_quantise(const F (&x)[8], uint32_t (&words)[2], float& scale) {
    constexpr int M = BITS == 8 ? 127 : 7;
    F top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = kv_abs_max(top, x[i]);
#pragma unroll
    for (int d = LANES / 2; d >= 1; d >>= 1) top = kv_abs_max(top, __shfl_xor_sync(0xffffffffu, top, d));
    scale = static_cast<float>(kv_divide(top, static_cast<F>(M)));
    words[0] = words[1] = 0;
    // x M / top by the inverse of top; where that comes near the middle between two codes (its error is below 2^-16 or 2^-44) the
    // quotient itself decides
    const bool sound = top > 0 && top < static_cast<F>(INFINITY);
    const F inverse = sound ? kv_divide(static_cast<F>(M), top) : static_cast<F>(0), near = static_cast<F>(0.5) - (sizeof(F) == 4 ? static_cast<F>(1e-4) : static_cast<F>(1e-9));
    const bool small = inverse > static_cast<F>(sizeof(F) == 4 ? 1e38 : 1e300);       // the inverse of a subnormal: every quotient itself
    // a quotient near such a middle is that of two large numbers, where x M would leave the type: both smaller, exactly
    const F down = sizeof(F) == 4 && top > static_cast<F>(1.2676506e30) ? static_cast<F>(0.00390625) : static_cast<F>(1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        F off;
        int code = kv_nearest(small ? static_cast<F>(0) : x[i] * inverse, off);
        if (sound && (small || fabs(off) > near)) code = kv_nearest(kv_divide(x[i] * down * static_cast<F>(M), top * down), off);
        if (!sound) code = 0;
        if constexpr (BITS == 8) words[i >> 2] |= static_cast<uint32_t>(code & 0xff) << (8 * (i & 3));
        else words[0] |= static_cast<uint32_t>(code + 8) << (4 * i);
    }
}

template <int BITS, int D>
__device__ __forceinline__ void kv_store_codes(void* pool, float* scales, int64_t vector, int lane, const uint32_t (&words)[2], float scale) {
    char* dst = static_cast<char*>(pool) + vector * (D * BITS / 8) + lane * BITS;
    if constexpr (BITS == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint32_t*>(dst) = words[0];
    if (lane == 0) scales[vector] = scale;
}

template <typename T, int BITS, int D, int ROWS>
__global__ void __launch_bounds__(kKvThreads, 4)
kv_append_kernel(const KvArgs p, const KvAppendArgs a) {
    // every row has warps of its own, all of which get their share of q, k and v
    constexpr int LANES = D / 8, kRowThreads = kKvThreads / ROWS, kGroups = kRowThreads / LANES, kAtOnce = 4;
    static_assert(kRowThreads % 32 == 0, "whole warps");
    __shared__ int s_start[kKvStarts + 1];
    __shared__ KvRow s_row[ROWS];
    __shared__ double2 s_turn[ROWS][BITS == 16 ? 1 : D / 2];      // cosine and sine
    __shared__ float2 s_turn_f[ROWS][D / 2];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS;
    kv_locate<ROWS>(p, row0, s_start, s_row);
    const int pairs = a.rotated / 2;
    for (int i = threadIdx.x; i < ROWS * pairs; i += kKvThreads) {
        const int r = i / pairs, j = i - r * pairs;
        const double turns = static_cast<double>(s_row[r].pos) * __ldg(a.turns + j);
        double sn, cs;
        sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
        cs *= a.magnitude;
        sn *= a.magnitude;
        s_turn_f[r][j] = make_float2(static_cast<float>(cs), static_cast<float>(sn));
        if constexpr (BITS != 16) s_turn[r][j] = make_double2(cs, sn);
    }
    __syncthreads();
    const int lane = threadIdx.x % LANES, group = threadIdx.x % kRowThreads / LANES;
    const int vectors = a.heads + 2 * p.kv_heads;
    const int d0 = lane * 8;
    // this lane's partner in the half layout: the same place of the other half of the rotated dimensions
    const int half_lanes = a.rotated / 16;
    const bool rotates = d0 < a.rotated, upper = lane >= half_lanes;
    const int partner = !rotates || a.interleaved ? lane : (upper ? lane - half_lanes : lane + half_lanes);
    const int pair0 = !rotates ? 0 : a.interleaved ? d0 / 2 : (upper ? d0 - pairs : d0);
    {
        const int r = threadIdx.x / kRowThreads;
        const KvRow at = s_row[r];
        if (at.pos < 0) return;                                   // the same for all of the row's warps
        const int64_t row = row0 + r;
        // the lane's dimensions are the same of every head, and so are its angles
        float2 turn_f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) turn_f[i] = rotates ? s_turn_f[r][a.interleaved ? pair0 + i / 2 : pair0 + i] : make_float2(1.0f, 0.0f);
#pragma unroll 1
        for (int first = 0; first < vectors; first += kAtOnce * kGroups) {
            uint4 loaded[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int vec = first + u * kGroups + group;
                loaded[u] = make_uint4(0, 0, 0, 0);
                if (vec < vectors) {
                    const T* src = vec < a.heads ? static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(vec) * D
                                   : vec < a.heads + p.kv_heads ? static_cast<const T*>(a.k) + row * a.k_stride + static_cast<int64_t>(vec - a.heads) * D
                                                                : static_cast<const T*>(a.v) + row * a.v_stride + static_cast<int64_t>(vec - a.heads - p.kv_heads) * D;
                    loaded[u] = *reinterpret_cast<const uint4*>(src + d0);
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                // whole warps go round together (the shuffles); a group without a vector holds zeros and stores nothing
                if (first + u * kGroups >= vectors) break;
                const int vec = first + u * kGroups + group;
                const bool is_q = vec < a.heads, is_k = !is_q && vec < a.heads + p.kv_heads;
                const int head = is_q ? vec : (is_k ? vec - a.heads : vec - a.heads - p.kv_heads);
                const bool live = vec < vectors && (is_q || at.place >= 0);
                const uint32_t own[4] = {loaded[u].x, loaded[u].y, loaded[u].z, loaded[u].w};
                uint32_t other[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) other[i] = __shfl_sync(0xffffffffu, own[i], partner, LANES);
                // x[i] of dimension d0 + i turned, in F
                auto turn = [&](auto angle, auto (&x)[8]) {
                    using F = std::remove_reference_t<decltype(x[0])>;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = KvType<T>::unpack(own[i]), o = KvType<T>::unpack(other[i]);
                        x[2 * i] = f.x;
                        x[2 * i + 1] = f.y;
                        const auto t0 = angle(2 * i), t1 = angle(2 * i + 1);
                        const F u0 = f.x, u1 = f.y, y0 = o.x, y1 = o.y;
                        if (!rotates) continue;
                        if (a.interleaved) {
                            x[2 * i] = u0 * t0.x - u1 * t0.y;
                            x[2 * i + 1] = u0 * t0.y + u1 * t0.x;
                        } else if (upper) {
                            x[2 * i] = y0 * t0.y + u0 * t0.x;
                            x[2 * i + 1] = y1 * t1.y + u1 * t1.x;
                        } else {
                            x[2 * i] = u0 * t0.x - y0 * t0.y;
                            x[2 * i + 1] = u1 * t1.x - y1 * t1.y;
                        }
                    }
                };
                auto angle_f = [&](int i) { return turn_f[i]; };
                auto store = [&](T* dst, const float (&x)[8]) {
                    *reinterpret_cast<uint4*>(dst) = make_uint4(KvType<T>::pack(x[0], x[1]), KvType<T>::pack(x[2], x[3]), KvType<T>::pack(x[4], x[5]),
                                                                KvType<T>::pack(x[6], x[7]));
                };
                const int64_t vector = at.place + static_cast<int64_t>(head) * p.page_size;
                if (is_q ? live : BITS == 16 && is_k && live) {
                    float x[8];
                    turn(angle_f, x);
                    store(is_q ? static_cast<T*>(a.q_out) + row * a.q_out_stride + static_cast<int64_t>(head) * D + d0 : static_cast<T*>(p.k) + vector * D + d0, x);
                }
                if constexpr (BITS == 16) {
                    if (!is_q && !is_k && live) *reinterpret_cast<uint4*>(static_cast<T*>(p.v) + vector * D + d0) = loaded[u];
                } else {
                    // a warp may hold vectors of several kinds: all its lanes go through the shuffles of both
                    uint32_t words[2];
                    float scale;
                    if (__any_sync(0xffffffffu, is_k && live)) {
                        double x[8];
                        turn([&](int i) { return s_turn[r][a.interleaved ? pair0 + i / 2 : pair0 + i]; }, x);
                        kv_quantise<BITS, LANES>(x, words, scale);
                        if (is_k && live) kv_store_codes<BITS, D>(p.k, p.k_scale, vector, lane, words, scale);
                    }
                    if (__any_sync(0xffffffffu, !is_q && !is_k && live)) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = KvType<T>::unpack(own[i]);
                            x[2 * i] = f.x;
                            x[2 * i + 1] = f.y;
                        }
                        kv_quantise<BITS, LANES>(x, words, scale);
                        if (!is_q && !is_k && live) kv_store_codes<BITS, D>(p.v, p.v_scale, vector, lane, words, scale);
                    }
                }
            }
        }
    }
}

template <typename O>
__device__ __forceinline__ void kv_store8(O* dst, const float (&x)[8]) {
    if constexpr (sizeof(O) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(KvType<O>::pack(x[0], x[1]), KvType<O>::pack(x[2], x[3]), KvType<O>::pack(x[4], x[5]),
                                                    KvType<O>::pack(x[6], x[7]));
    }
}

// T: type of a 16-bit cache (any for codes); O: type of the rows
template <typename T, int BITS, int D, typename O, int ROWS>
__global__ void __launch_bounds__(kKvThreads)
kv_read_kernel(const KvArgs p, O* __restrict__ k_out, O* __restrict__ v_out) {
    constexpr int LANES = D / 8, kRowThreads = kKvThreads / ROWS, kGroups = kRowThreads / LANES;
    __shared__ int s_start[kKvStarts + 1];
    __shared__ KvRow s_row[ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS;
    kv_locate<ROWS>(p, row0, s_start, s_row);
    const int lane = threadIdx.x % LANES, group = threadIdx.x % kRowThreads / LANES, vectors = 2 * p.kv_heads;
    const int r = threadIdx.x / kRowThreads;                      // every row has threads of its own
    const KvRow at = s_row[r];
    if (at.place < 0) return;
    constexpr int kAtOnce = 4;
#pragma unroll 1
    for (int first = group; first < vectors; first += kAtOnce * kGroups) {
        uint4 loaded[kAtOnce];                                    // 16, 8 or 4 bytes of it
        float scale[kAtOnce];
        O* dst[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int vec = first + u * kGroups;
            const bool is_k = vec < p.kv_heads;
            const int head = is_k ? vec : vec - p.kv_heads;
            O* out = is_k ? k_out : v_out;
            dst[u] = vec < vectors && out != nullptr ? out + ((row0 + r) * p.kv_heads + head) * D + lane * 8 : nullptr;
            scale[u] = 0.0f;
            if (dst[u] == nullptr) continue;
            const int64_t vector = at.place + static_cast<int64_t>(head) * p.page_size;
            const char* src = static_cast<const char*>(is_k ? p.k : p.v) + vector * (D * BITS / 8) + lane * BITS;
            if constexpr (BITS == 16) loaded[u] = __ldcs(reinterpret_cast<const uint4*>(src));
            else {
                if constexpr (BITS == 8) { const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src)); loaded[u].x = w.x; loaded[u].y = w.y; }
                else loaded[u].x = __ldcs(reinterpret_cast<const uint32_t*>(src));
                scale[u] = __ldg((is_k ? p.k_scale : p.v_scale) + vector);
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if (dst[u] == nullptr) continue;
            float x[8];
            if constexpr (BITS == 16) {
                const uint32_t words[4] = {loaded[u].x, loaded[u].y, loaded[u].z, loaded[u].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = KvType<T>::unpack(words[i]);
                    x[2 * i] = f.x;
                    x[2 * i + 1] = f.y;
                }
            } else if constexpr (BITS == 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = scale[u] * static_cast<float>(static_cast<int8_t>((i < 4 ? loaded[u].x : loaded[u].y) >> (8 * (i & 3))));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = scale[u] * static_cast<float>(static_cast<int>((loaded[u].x >> (4 * i)) & 15u) - 8);
            }
            kv_store8(dst[u], x);
        }
    }
}

// One row a CTA while that leaves SMs free: a short call is the latency of one row.  Eight (four appended) rows share the search
// and fill the CTA's threads where there are many.
template <int MANY>
bool kv_many_rows(int64_t rows) { return rows >= static_cast<int64_t>(MANY) * sm_count(); }

template <typename T, int BITS, int D>
cudaError_t launch_append(const KvArgs& p, const KvAppendArgs& a, cudaStream_t stream) {
    if (kv_many_rows<4>(p.rows))
        return launch_dependent(kv_append_kernel<T, BITS, D, 4>, dim3(static_cast<unsigned>((p.rows + 3) / 4)), dim3(kKvThreads), 0, stream, p, a);
    return launch_dependent(kv_append_kernel<T, BITS, D, 1>, dim3(static_cast<unsigned>(p.rows)), dim3(kKvThreads), 0, stream, p, a);
}

template <typename T, int BITS, int D, typename O>
cudaError_t launch_read(const KvArgs& p, void* k, void* v, cudaStream_t stream) {
    O* ko = static_cast<O*>(k);
    O* vo = static_cast<O*>(v);
    if (kv_many_rows<8>(p.rows))
        return launch_dependent(kv_read_kernel<T, BITS, D, O, 8>, dim3(static_cast<unsigned>((p.rows + 7) / 8)), dim3(kKvThreads), 0, stream, p, ko, vo);
    return launch_dependent(kv_read_kernel<T, BITS, D, O, 1>, dim3(static_cast<unsigned>(p.rows)), dim3(kKvThreads), 0, stream, p, ko, vo);
}

template <typename T, int BITS, int D>
cudaError_t launch_read_out(const KvArgs& p, int out_dtype, void* k, void* v, cudaStream_t stream) {
    if (out_dtype == kF32) return launch_read<T, BITS, D, float>(p, k, v, stream);
    if (out_dtype == kF16) return launch_read<T, BITS, D, __half>(p, k, v, stream);
    return launch_read<T, BITS, D, __nv_bfloat16>(p, k, v, stream);
}

}  // namespace

bool kv_tensor_maps(const KvArgs& p, int most, CUtensorMap* k_map, CUtensorMap* v_map, int* box_rows) {
    using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn encode = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            ptr = nullptr;
        return reinterpret_cast<EncodeFn>(ptr);
    }();
    const int64_t vectors = p.pages * p.kv_heads * p.page_size;
    const int rows = std::min(most, p.page_size & -p.page_size);
    if (!encode || rows < 8 || vectors > INT32_MAX) return false;       // eight rows are an atom of the swizzle
    if (p.bits != 16 && ((reinterpret_cast<uintptr_t>(p.k_scale) | reinterpret_cast<uintptr_t>(p.v_scale)) & 15u)) return false;     // their scales are copied in bulk
    const cuuint32_t width = static_cast<cuuint32_t>(p.head_dim * p.bits / 8), box_width = std::min(width, 128u);
    const cuuint64_t dims[2] = {width, static_cast<cuuint64_t>(vectors)}, strides[1] = {width};
    const cuuint32_t box[2] = {box_width, static_cast<cuuint32_t>(rows)}, elem[2] = {1, 1};
    const CUtensorMapSwizzle swizzle = box_width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : box_width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    for (int kind = 0; kind < 2; ++kind)
        if (encode(kind ? v_map : k_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, kind ? p.v : p.k, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    *box_rows = rows;
    return true;
}

cudaError_t launch_kv_append(const KvArgs& p, const KvAppendArgs& a, cudaStream_t stream) {
#define B200_KV_CASE(T, BITS, D) \
    if (p.bits == BITS && p.head_dim == D) return launch_append<T, BITS, D>(p, a, stream);
#define B200_KV_CASES(T)                                                      \
    B200_KV_CASE(T, 16, 128) B200_KV_CASE(T, 16, 64) B200_KV_CASE(T, 8, 128) \
    B200_KV_CASE(T, 8, 64) B200_KV_CASE(T, 4, 128) B200_KV_CASE(T, 4, 64)
    if (p.dtype == kF16) { B200_KV_CASES(__half) }
    else { B200_KV_CASES(__nv_bfloat16) }
#undef B200_KV_CASES
#undef B200_KV_CASE
    return cudaErrorInvalidValue;
}

cudaError_t launch_kv_read(const KvArgs& p, int out_dtype, void* k, void* v, cudaStream_t stream) {
    if (p.bits == 16) {
        if (p.dtype == kF16) return p.head_dim == 128 ? launch_read_out<__half, 16, 128>(p, out_dtype, k, v, stream) : launch_read_out<__half, 16, 64>(p, out_dtype, k, v, stream);
        return p.head_dim == 128 ? launch_read_out<__nv_bfloat16, 16, 128>(p, out_dtype, k, v, stream) : launch_read_out<__nv_bfloat16, 16, 64>(p, out_dtype, k, v, stream);
    }
    if (p.bits == 8) return p.head_dim == 128 ? launch_read_out<__half, 8, 128>(p, out_dtype, k, v, stream) : launch_read_out<__half, 8, 64>(p, out_dtype, k, v, stream);
    return p.head_dim == 128 ? launch_read_out<__half, 4, 128>(p, out_dtype, k, v, stream) : launch_read_out<__half, 4, 64>(p, out_dtype, k, v, stream);
}

}  // namespace b200exl3
