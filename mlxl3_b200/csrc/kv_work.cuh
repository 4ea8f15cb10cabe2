// How the attention kernels over the paged cache share out their work.  A segment is up to ROWS rows (token-major, then head) of one
// sequence and key head -- the query heads that share a key head are rows of one product -- and its keys come in blocks of KEYS.  The
// blocks of all segments, one after the other, are dealt out to the CTAs of one wave in equal runs: ragged lengths, few sequences
// and few heads all keep every SM busy, and since the lengths are read on the device a recorded call serves growing sequences.  A
// segment counts OVER units before its first block, for what its beginning and its end cost.
// A CTA that holds a whole segment stores it; CTAs that share one leave (maximum, sum, unnormalised rows) and the last to arrive joins
// the parts in the order of the keys.
#pragma once

#include <cuda.h>

#include "kv.cuh"
#include "tcgen05.cuh"

namespace b200exl3 {

struct KvSegment {
    int first, last;       // tokens of the segment
    int low, blocks;       // first key of the first block; blocks (one at least: rows that see nothing are stored too)
    int key0, key1;        // visible keys
};

// Keys that the row at `position` sees: first .. end - 1.  A sequence with more rows than tokens begins before position 0; any window.
__device__ __forceinline__ int kv_seen_end(int position, int capacity) { return min(max(position + 1, 0), capacity); }
__device__ __forceinline__ int kv_seen_first(int position, int window) { return window > 0 ? max(max(position + 1, 0) - window, 0) : 0; }

// Sequences whose first rows and lengths a CTA keeps in shared memory; more are read where they are.
template <int CAP>
struct KvTable {
    int start[CAP + 1], length[CAP];
};

template <int ROWS, int KEYS, int OVER>
struct KvWork {
    const KvArgs& p;
    const KvAttentionArgs& a;
    const int* start;      // [batch + 1], [batch]
    const int* length;
    int group, capacity;

    template <int CAP>
    __device__ __forceinline__ KvWork(const KvArgs& p_, const KvAttentionArgs& a_, KvTable<CAP>& table) : p(p_), a(a_) {
        group = a.heads / p.kv_heads;
        capacity = static_cast<int>(min(p.table_width * static_cast<int64_t>(p.page_size), static_cast<int64_t>(kKvMaxTokens)));
        start = p.row_start;
        length = p.length;
        if (p.batch <= CAP) {
            for (int i = threadIdx.x; i <= p.batch; i += blockDim.x) {
                table.start[i] = __ldg(p.row_start + i);
                if (i < p.batch) table.length[i] = __ldg(p.length + i);
            }
            __syncthreads();
            start = table.start;
            length = table.length;
        }
    }
    __device__ __forceinline__ KvSeq seq(int b) const {
        KvSeq s;
        s.first_row = kv_clamp_row(p, start[b]);
        s.n = max(0, kv_clamp_row(p, start[b + 1]) - s.first_row);
        s.first_pos = kv_clamp_length(length[b]) - s.n;
        return s;
    }
    // rows of a sequence that this kernel takes: all or none
    __device__ __forceinline__ int rows_of(const KvSeq& s) const {
        const int rows = min(s.n, a.max_new) * group;
        return rows >= a.least_rows && rows <= a.most_rows ? rows : 0;
    }
    // Keys that some row of a sequence sees end here; whether its rows see different keys; keys that all rows of a segment see
    __device__ __forceinline__ int any_end(const KvSeq& s) const { return min(s.first_pos + min(s.n, a.max_new), capacity); }
    __device__ __forceinline__ bool several(const KvSeq& s) const { return min(s.n, a.max_new) > 1; }
    __device__ __forceinline__ int all_first(const KvSeq& s, const KvSegment& g) const { return kv_seen_first(s.first_pos + g.last, a.window); }
    __device__ __forceinline__ int all_end(const KvSeq& s, const KvSegment& g) const { return kv_seen_end(s.first_pos + g.first, capacity); }
    __device__ __forceinline__ int tiles_of(const KvSeq& s) const { return (rows_of(s) + ROWS - 1) / ROWS; }
    __device__ __forceinline__ KvSegment segment(const KvSeq& s, int tile) const {
        KvSegment g;
        const int rows = min(s.n, a.max_new) * group;
        g.first = tile * ROWS / group;
        g.last = (min(rows, (tile + 1) * ROWS) - 1) / group;
        g.key1 = kv_seen_end(s.first_pos + g.last, capacity);
        g.key0 = kv_seen_first(s.first_pos + g.first, a.window);
        g.low = g.key0 / KEYS * KEYS;
        g.blocks = max(1, (g.key1 - g.low + KEYS - 1) / KEYS);
        return g;
    }
    // units of all row tiles of a sequence, for one key head; LANES neighbouring lanes count together
    template <int LANES>
    __device__ __forceinline__ int64_t units_of(const KvSeq& s) const {
        int64_t sum = 0;
        const int tiles = tiles_of(s);
        for (int t = LANES > 1 ? static_cast<int>(threadIdx.x) % LANES : 0; t < tiles; t += LANES) sum += OVER + segment(s, t).blocks;
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        return sum;
    }
};

// Walks the blocks of a run: [sequence][key head][row tile][block].  The blocks of the segment at hand are block .. end - 1.
template <int ROWS, int KEYS, int OVER>
struct KvCursor {
    using Work = KvWork<ROWS, KEYS, OVER>;
    int b, head, tile, block, end;
    int64_t base, left;    // unit at which the segment begins; units of the run behind this segment
    KvSeq seq;
    KvSegment seg;

    // the segment at hand, entered at its unit `at`
    __device__ __forceinline__ void enter(int64_t at) {
        const int64_t units = min(seg.blocks + OVER - at, left);
        left -= units;
        block = static_cast<int>(max(at - OVER, static_cast<int64_t>(0)));
        end = static_cast<int>(max(at + units - OVER, static_cast<int64_t>(0)));
    }
    // the next segment of the run that has blocks in it; false: the run is at its end
    __device__ __forceinline__ bool next_segment(const Work& w) {
        while (left > 0) {
            base += seg.blocks + OVER;
            if (++tile == w.tiles_of(seq)) {
                tile = 0;
                if (++head == w.p.kv_heads) {
                    head = 0;
                    do {
                        if (++b >= w.p.batch) return false;
                        seq = w.seq(b);
                    } while (w.rows_of(seq) == 0);
                }
            }
            seg = w.segment(seq, tile);
            enter(0);
            if (block < end) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool step(const Work& w) { return ++block < end || next_segment(w); }
};

__device__ __forceinline__ int64_t kv_quotient(int64_t a, int64_t b) {      // of non-negative numbers
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// `total` units dealt out to `ctas` CTAs: `each` to every one, one more to the first `more`.
struct KvRun {
    int64_t total, each;
    int ctas, more;

    __device__ __forceinline__ void deal(int64_t total_, int grid) {
        total = total_;
        ctas = static_cast<int>(min(static_cast<int64_t>(grid), total));
        each = ctas > 0 ? kv_quotient(total, ctas) : 0;
        more = static_cast<int>(total - each * ctas);
    }
    __device__ __forceinline__ int64_t first(int cta) const { return cta * each + min(cta, more); }
    // the CTA that holds unit u
    __device__ __forceinline__ int cta_of(int64_t u) const {
        const int64_t longer = more * (each + 1);
        return static_cast<int>(u < longer ? kv_quotient(u, each + 1) : more + kv_quotient(u - longer, each));
    }
};

// Finds this CTA's run; every thread of the block calls it.  Workers of LANES threads (1, or 32: sequences of many row tiles) count a
// slice of the sequences each; the one whose slice holds the first unit writes the place.  Returns false where there is nothing to do.
template <int THREADS, int LANES, int ROWS, int KEYS, int OVER>
__device__ __forceinline__ bool kv_find_run(const KvWork<ROWS, KEYS, OVER>& w, int64_t (&s_sum)[THREADS / LANES + 1],
                                            KvCursor<ROWS, KEYS, OVER>& s_cursor, KvRun& run) {
    constexpr int kWorkers = THREADS / LANES;
    static_assert(LANES == 1 || LANES == 32, "threads or warps");
    const int worker = threadIdx.x / LANES, sub = threadIdx.x % LANES;
    const int slice = (w.p.batch + kWorkers - 1) / kWorkers;
    const int b0 = min(w.p.batch, worker * slice), b1 = min(w.p.batch, b0 + slice);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += w.template units_of<LANES>(w.seq(b)) * w.p.kv_heads;
    if (sub == 0) s_sum[worker] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {                                       // exclusive sums
        int64_t carry = 0;
        for (int i0 = 0; i0 < kWorkers; i0 += 32) {
            const int i = i0 + static_cast<int>(threadIdx.x);
            const int64_t own = i < kWorkers ? s_sum[i] : 0;
            int64_t upto = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
                if (static_cast<int>(threadIdx.x) >= d) upto += o;
            }
            if (i < kWorkers) s_sum[i] = carry + upto - own;
            carry += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (threadIdx.x == 0) s_sum[kWorkers] = carry;
    }
    __syncthreads();
    run.deal(s_sum[kWorkers], gridDim.x);
    if (static_cast<int>(blockIdx.x) >= run.ctas) return false;
    const int64_t before = s_sum[worker], u0 = run.first(blockIdx.x);
    if (before <= u0 && u0 < before + mine) {
        int64_t left = u0 - before;
        KvCursor<ROWS, KEYS, OVER> c;
        for (int b = b0; b < b1; ++b) {
            c.seq = w.seq(b);
            const int64_t per_head = w.template units_of<LANES>(c.seq);
            if (left >= per_head * w.p.kv_heads) {
                left -= per_head * w.p.kv_heads;
                continue;
            }
            c.b = b;
            c.head = static_cast<int>(kv_quotient(left, per_head));
            left -= c.head * per_head;
            for (c.tile = 0;; c.tile += LANES) {
                const int tile = c.tile + sub, tiles = w.tiles_of(c.seq);
                const int n = tile < tiles ? OVER + w.segment(c.seq, tile).blocks : 0;
                if constexpr (LANES == 1) {
                    if (left < n) break;
                    left -= n;
                } else {
                    int upto = n;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const int o = __shfl_up_sync(0xffffffffu, upto, d);
                        if (sub >= d) upto += o;
                    }
                    const unsigned int past = __ballot_sync(0xffffffffu, left < upto);
                    if (past != 0) {
                        const int lane = __ffs(past) - 1;
                        left -= __shfl_sync(0xffffffffu, upto - n, lane);
                        c.tile += lane;
                        break;
                    }
                    left -= __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            c.seg = w.segment(c.seq, c.tile);
            c.base = u0 - left;
            c.left = run.first(blockIdx.x + 1) - u0;
            c.enter(left);
            if (c.block == c.end && !c.next_segment(w)) c.end = c.block;     // the run begins before a segment's first block
            break;
        }
        if (sub == 0) s_cursor = c;
    }
    __syncthreads();
    return s_cursor.block < s_cursor.end;
}

__device__ __forceinline__ float exp2_fast(float x) {             // 2 ulp; exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / sum of a row; a row that sees nothing is zero
__device__ __forceinline__ float kv_inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

// Probabilities are rounded to 16 bits for the second product as 2^(s + lift - m), where m bounds the row's scores so far to within 8.  fp16:
// from 2^7 to 2^15, so that what lies 2^21 below the largest still has all its bits, and all of a long context's small ones add up (2^-32
// of the largest at worst).  bf16, whose range is that of fp32: far below one, so that sums of the type's largest values stay finite.
template <typename M> constexpr float kLift = 7.0f;
template <> constexpr float kLift<__nv_bfloat16> = -32.0f;
// Over a quantised cache it is w = 2^(s + lift - m) vs, the probability times the value's scale, and m bounds s + log2 vs over the keys that
// the row itself sees: a rounding costs 2^-11 of a term, or 2^-32 of the row's largest one, whatever scales other keys have.  The sum of
// the probabilities has 2^(s + lift - m).  So that it fits fp32 for scales at the ends of its range too, they enter as vs / 2^16, and
// their logarithm is not taken below -88: sums reach 2^(88 + 15) a key, and a largest term of scale 2^125 (4-bit bf16) is 2^-102.
// Scales below 2^-93 lose bits, those below 2^-104 are zero.
constexpr float kScaleUnit = 65536.0f;
__device__ __forceinline__ float kv_scale_log(float vs) {         // of a scale in that unit; NaN: the least
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(vs));
    return fmaxf(y, -88.0f);
}

// The power of two that brings a row's largest magnitude to [1, 2), and its inverse, in two factors each: all of them are normal numbers.
struct KvPower {
    float down0, down1, up0, up1;
    __device__ __forceinline__ explicit KvPower(float top) {
        const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127, half = e >> 1;        // -127 for 0
        down0 = power(-half);
        down1 = power(half - e);
        up0 = power(half);
        up1 = power(e - half);
    }
    static __device__ __forceinline__ float power(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
};

__device__ __forceinline__ void copy16_fill(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_fill(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void shared_load4(uint32_t src, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Where a 16-byte chunk of a tile's row lies, as the tensor copies put it: pieces of up to 128 bytes of all rows, one after the other; in
// a piece rows of 128 bytes swap their chunks by the row's number, shorter ones by the number of the 128 bytes they are in, so that eight
// rows' same chunk uses all banks.
template <int CHUNKS, int KEYS>
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
    constexpr int kPiece = CHUNKS >= 8 ? 8 : CHUNKS, kShift = CHUNKS >= 8 ? 0 : (CHUNKS == 4 ? 1 : 2);
    return static_cast<uint32_t>((chunk / kPiece * KEYS + row) * kPiece + ((chunk % kPiece) ^ ((row >> kShift) & (kPiece - 1)))) * 16;
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

// `rows` rows of the pool, 128 bytes of each at most (column c0 on), into shared memory by the tensor-copy unit
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int c0, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(smem_addr(bar)), "r"(c0), "r"(row) : "memory");
}

// Host: the pool's vectors as rows of a 2-D tensor, copied in boxes of box_rows rows of up to 128 bytes, swizzled over the row's width.
// False where there are no such copies; box_rows is the largest power of two that divides the page size, at most `most`.
bool kv_tensor_maps(const KvArgs& p, int most, CUtensorMap* k_map, CUtensorMap* v_map, int* box_rows);

}  // namespace b200exl3
