// Softmax attention of a step's rows over a paged cache: one token of a sequence, a chunk, a whole prompt, sequences of each kind in one
// launch.
//
//   out = sum_j softmax_j(scale q . k_j [, sink]) v_j   over the positions j up to the row's own, the last `window` of them where there is one
//
// A tile is 16 or 128 packed rows (row of the sequence, head of the group) of one kv head; the tiles of all sequences are counted off
// from `starts` by every wave.  Running maximum and sum in 32 bits, in powers of two.
#include "paged.hpp"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

typedef _Float16 lh_f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f;

// Positions of a step of the kernel for many rows, by the padded columns of a head.
__host__ __device__ constexpr uint32_t tile_step(uint32_t columns) { return columns <= 128 ? 64 : 32; }

// n / d for n below 2^31 by a product and a shift (a division is some 30 instructions, one waiting for the other, and a launch of a few microseconds has a
// dozen): with s = ceil(log2 d) and m = ceil(2^(31 + s) / d), m d exceeds 2^(31 + s) by less than 2^s, which n times is less than 2^(31 + s).
struct Divisor {
    uint32_t d, m, shift;
    Divisor() = default;
    explicit Divisor(uint32_t by) : d(by) {
        uint32_t s = 0;
        while ((1ull << s) < by) s++;
        shift = 31 + s;
        m = (uint32_t)(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (uint32_t)((uint64_t)n * m >> shift); }
};

struct PagedArgs {
    const void *q, *keys, *values;
    void* out;
    const float* sink;         // [heads], may be null
    float* partial;            // records of (D + 4) values a row, a part's by Tile::record_of: unnormalised sums, maximum, sum of weights
    PagedPlan plan;
    uint64_t q_ld, out_ld;
    uint32_t max_rows, heads, kv_heads, dim, window, capacity;     // capacity: positions from there on are not seen
    uint32_t most, least, fill, share, coarse, fixed;              // how tiles are cut (chunk_of): steps of a tile at most and of a part at least; workgroups wanted,
                                                                   // and of a kv head; what the sum is shifted by; nothing to measure
    uint32_t parts;                                                // of all tiles at most
    uint32_t records, rows_kept;                                   // records of a kv head that the workspace takes; rows of one
    uint32_t stream;                                               // the caches may be more than is worth keeping near the chip
    uint32_t q_wide, out_wide;                                     // rows, heads and their ends at 16 bytes
    uint32_t q_plain;                                              // nothing to be done to the queries as they are loaded
    float scale2;              // of the products, in powers of two; > 0
    uint32_t negative, nothing;                                    // the scale is below zero, or zero: in the queries
    Divisor group, by_heads;                                       // query heads of a kv head; kv heads
};

// The sum over this lane and the ones before it.
__device__ __forceinline__ uint32_t sum_up_to(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // row_shr:1, 2, 4, 8, row_bcast:15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xE, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xC, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// n / d rounded down, or one less: by the reciprocal (good to 2^-22), for quotients below 2^20.
__device__ __forceinline__ uint32_t about(uint32_t n, uint32_t d) {
    const uint32_t q = (uint32_t)((float)n * __builtin_amdgcn_rcpf((float)d));
    return q * d > n ? q - 1 : q;
}
__device__ __forceinline__ uint32_t whole(uint32_t n, uint32_t d) {
    const uint32_t q = about(n, d);
    return n - q * d >= d ? q + 1 : q;
}

// What a lane's sequence has: tiles, and steps of positions that each may take at most.
struct Load { uint32_t first, all, length, tiles, steps; };
template <uint32_t ROWS, uint32_t STEP>
__device__ __forceinline__ Load load_of(const PagedArgs& a, uint32_t s) {
    Load c;
    const uint32_t some = min(s, a.plan.sequences - 1);       // (loads without branches go out together)
    c.first = a.plan.starts[some];
    c.length = a.plan.lengths[some];
    const uint32_t end = a.plan.starts[some + 1];
    const bool on = s < a.plan.sequences && end > c.first && end <= a.plan.rows;
    c.all = on ? end - c.first : 0u;
    c.tiles = (uint32_t)(((uint64_t)min(c.all, a.max_rows) * a.group.d + ROWS - 1) / ROWS);
    c.steps = on ? min((min(c.length, a.capacity) + STEP - 1) / STEP, a.most) : 0u;
    return c;
}

// Steps of a part: what all tiles have to do over the workgroups wanted, so that a long sequence among short ones is cut and short ones alone are not, whatever bound the
// call gives for their lengths (64 tokens at 4000 of a call for up to 131072: parts by the bound 313 us, so 171; 256 at 1000 653 and 174).  The exception is a call whose
// bounds fill the chip with tiles of at most 128 steps: nothing of it is cut (cut(), where it is measured).  Where there are few tiles,
// equal ones make a whole number of parts.  It costs every workgroup two scans and a reciprocal, 0.2 us, and 5 with a thousand sequences (1024 at 1000 in a call for up to 16384
// 658 -> 694 us).  All kernels of a call find the same.
//   The sum is of steps shifted by `coarse` and rounded up, which lets it fit.  The chunk is at least what all have over `share`: so the parts of all tiles are at most
//   `share` more than there are tiles, and, a tile in parts having more than a chunk, those of such tiles at most twice `share`.
template <uint32_t ROWS, uint32_t STEP>
__device__ __forceinline__ uint32_t chunk_of(const PagedArgs& a, uint32_t lane, Load& c, uint32_t& longest) {
    if (a.fixed) {
        if (a.plan.sequences <= 64) c = load_of<ROWS, STEP>(a, lane);
        longest = a.most;
        return a.least;
    }
    uint32_t tiles = 0, work = 0;
    longest = 0;
#pragma unroll 4
    for (uint32_t s0 = 0; s0 < a.plan.sequences; s0 += 64) {
        c = load_of<ROWS, STEP>(a, s0 + lane);
        tiles += c.tiles;
        longest = max(longest, c.steps);
        work += (uint32_t)(((uint64_t)c.tiles * c.steps + (1ull << a.coarse) - 1) >> a.coarse);
    }
    tiles = __builtin_amdgcn_readlane(sum_up_to(tiles), 63);
    work = __builtin_amdgcn_readlane(sum_up_to(work), 63);
    const uint64_t units = (uint64_t)tiles * a.kv_heads;
    // (a reciprocal's error cannot take the quotient over a whole number, nor the chunk below what it has to be)
    const float each = units >= a.fill ? 0.0f : __builtin_truncf((float)a.fill * __builtin_amdgcn_rcpf((float)max((uint32_t)units, 1u)) * 1.00001f);
    const float parts = units >= a.fill ? (float)a.share : max((float)tiles, 1.0f) * each;
    const uint32_t steps = (uint32_t)((float)work * __builtin_amdgcn_rcpf(parts) * 1.00001f) + 1;
    return max((uint32_t)min((uint64_t)steps << a.coarse, (uint64_t)a.most), a.least);
}

// A tile of a sequence: its rows row0 .. row0 + count - 1 of the packed ones; and part `split` of it.
struct Tile {
    int sequence;
    uint32_t row0, count, first;    // first: the sequence's first row in q
    int64_t begin;                  // position of the sequence's first row
    uint32_t split, parts, chunk;   // parts: at most
    uint32_t record;                // records of a kv head before its own, where it has several parts
    // The first record for kv head g; its parts' follow.
    __device__ __forceinline__ size_t record_of(const PagedArgs& a, uint32_t g) const { return (size_t)record * a.kv_heads + (size_t)g * parts; }
};
// Part n of all tiles, JOIN: tile n of those in parts.  All lanes get the same; sequence -1 behind the last.  A sequence's tiles of the same part follow each other, so
// that those that read the same pages at the same time are on different XCDs (on one, where the number of parts was a multiple of two, they waited for each
// other: 64 rows at 8000 25.1 us, 20.4 so; 1000 rows of 8 heads over 4 of 128 in f32 54 and 44).
template <uint32_t ROWS, uint32_t STEP, bool JOIN>
__device__ __forceinline__ Tile tile_of(const PagedArgs& a, uint32_t n, uint32_t lane) {
    const uint32_t R = a.group.d;
    Tile r{-1, 0, 0, 0, 0, 0, 1, 0, 0};
    Load own;
    uint32_t longest, before = 0, records = 0;
    r.chunk = chunk_of<ROWS, STEP>(a, lane, own, longest);
    if (JOIN && !__any(longest > r.chunk)) return r;
    // whether it is of the 64 sequences from s0 on
    const auto found = [&](const Load& c, uint32_t s0) __attribute__((always_inline)) {
        const uint32_t parts = max(about(c.steps + r.chunk - 1, r.chunk), 1u), all = c.tiles * parts, kept = parts > 1 ? all : 0u, size = JOIN ? (parts > 1 ? c.tiles : 0u) : all;
        const uint32_t sum = sum_up_to(size), kept_sum = sum_up_to(kept);
        const uint64_t behind = __ballot(before + sum > n);
        if (!behind) {
            before += __builtin_amdgcn_readlane(sum, 63);
            records += __builtin_amdgcn_readlane(kept_sum, 63);
            return false;
        }
        const int at = __builtin_ctzll(behind);
        const uint32_t brought = __builtin_amdgcn_readlane(c.all, at), rows = min(brought, a.max_rows) * R;
        r.sequence = s0 + at;
        r.first = __builtin_amdgcn_readlane(c.first, at);
        r.parts = __builtin_amdgcn_readlane(parts, at);
        const uint32_t in = n - before - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(size, at)), tiles = __builtin_amdgcn_readlane(c.tiles, at);
        r.split = JOIN || r.parts == 1 ? 0u : whole(in, tiles);
        const uint32_t i = in - r.split * tiles;
        r.record = records + (__builtin_amdgcn_readlane(kept_sum, at) - __builtin_amdgcn_readlane(kept, at)) + i * r.parts;
        if (i >= tiles || (r.parts > 1 && r.record + r.parts > a.records)) r.sequence = -1;      // (only where starts do not ascend: the sums say nothing then)
        r.row0 = i * ROWS;
        r.count = min(ROWS, rows - r.row0);
        r.begin = (int64_t)(uint32_t)__builtin_amdgcn_readlane(c.length, at) - brought;
        return true;
    };
    if (a.plan.sequences <= 64) {
        found(own, 0);
        return r;
    }
    for (uint32_t s0 = 0; s0 < a.plan.sequences; s0 += 256) {
        const Load c[4] = {load_of<ROWS, STEP>(a, s0 + lane), load_of<ROWS, STEP>(a, s0 + 64 + lane), load_of<ROWS, STEP>(a, s0 + 128 + lane), load_of<ROWS, STEP>(a, s0 + 192 + lane)};
        if (found(c[0], s0) || found(c[1], s0 + 64) || found(c[2], s0 + 128) || found(c[3], s0 + 192)) return r;
    }
    return r;
}

// Positions lo .. hi - 1 are seen by a sequence's row `row`.
struct Seen { uint32_t lo, hi; };
__device__ __forceinline__ Seen seen_by(const PagedArgs& a, const Tile& t, uint32_t row) {
    const int64_t p = t.begin + row, cap = a.capacity;
    Seen s;
    s.hi = (uint32_t)min(max(p + 1, (int64_t)0), cap);
    s.lo = a.window ? (uint32_t)min(max(p + 1 - a.window, (int64_t)0), cap) : 0u;
    return s;
}

// The part of a tile's positions lo .. hi - 1 that split z takes, in steps of STEP; `used` splits have any.
struct Part { uint32_t begin, end, used; };
template <uint32_t STEP>
__device__ __forceinline__ Part part_of(const Tile& t, uint32_t lo, uint32_t hi, uint32_t z) {
    const uint32_t b0 = lo / STEP, b1 = max((hi + STEP - 1) / STEP, b0), n = b1 - b0;
    const uint32_t used = t.parts == 1 ? 1u : min(max(about(n + t.chunk - 1, t.chunk), 1u), t.parts);
    uint32_t per = n;
    if (used > 1) {
        per = about(n + used - 1, used) + (n >> 18);
        per += per * used < n;
    }
    return Part{min(b0 + z * per, b1), min(b0 + (z + 1) * per, b1), used};
}

// A wave's view of its sequence's row of the table: 64 entries at a time, one a lane.
struct Pages {
    const uint32_t* row;
    uint32_t blocks;                // entries that the wave may need
    uint32_t held, entry;           // entries held .. held + 63
    uint64_t there;                 // which of them are pages of the pool, or not needed
    __device__ __forceinline__ void ask(const PagedPlan& p, uint32_t from, uint32_t lane) {
        held = from;
        entry = from + lane < min(blocks, p.table_ld) ? row[from + lane] : 0xFFFFFFFFu;
    }
    __device__ __forceinline__ void settle(const PagedPlan& p, uint32_t lane) { there = __ballot(held + lane >= blocks || entry < p.pages); }
    __device__ __forceinline__ void load(const PagedPlan& p, uint32_t from, uint32_t lane) { ask(p, from, lane); settle(p, lane); }
    __device__ __forceinline__ void reach(const PagedPlan& p, uint32_t block, uint32_t lane) { if (block - held >= 64) load(p, block, lane); }
    // of a block that is held: whether it is there, and its page, or some page
    __device__ __forceinline__ bool has(uint32_t block) const { return there >> (block - held) & 1; }
    __device__ __forceinline__ uint32_t of(const PagedPlan& p, uint32_t block) const {
        const uint32_t pg = __builtin_amdgcn_readlane(entry, block - held);
        return pg < p.pages ? pg : 0u;
    }
};

template <int DT>
__device__ __forceinline__ lh_f32x4 product(u32x4 x, u32x4 y, lh_f32x4 c) {
    if constexpr (DT == kF16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lh_f16x8, x), __builtin_bit_cast(lh_f16x8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lh_bf16x8, x), __builtin_bit_cast(lh_bf16x8, y), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == kF16) {                               // (two roundings put together are three instructions)
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
    } else return lh_pack_bf(a, b);
}
template <int DT>
__device__ __forceinline__ float low(uint32_t x) { return element_value<DT>((element_t<DT>)(x & 0xFFFFu)); }
template <int DT>
__device__ __forceinline__ float high(uint32_t x) { return element_value<DT>((element_t<DT>)(x >> 16)); }

template <bool STREAM>
__device__ __forceinline__ u32x4 load16(const void* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(static_cast<const u32x4*>(p));
    else return *static_cast<const u32x4*>(p);
}
// N dwords from an address that is a multiple of their largest power of two
template <bool STREAM, int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&x)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) { const u32x4 v = load16<STREAM>((const char*)p + 4 * i); x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w; }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) { const uint2 v = *reinterpret_cast<const uint2*>((const char*)p + 4 * i); x[i] = v.x; x[i + 1] = v.y; }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = *reinterpret_cast<const uint32_t*>((const char*)p + 4 * i);
    }
}

// A lane's N pieces of 16 bytes of the query at q_at, the first at column d, `apart` columns from one to the next; zeros behind the head's
// end.  The scale's sign goes into them.  All loads are on their way together.
template <int DT, int N>
__device__ __forceinline__ void load_query(const PagedArgs& a, uint64_t q_at, uint32_t d, uint32_t apart, u32x4 (&x)[N]) {
    typedef element_t<DT> B;
    constexpr uint32_t n = 16 / sizeof(B);
    const B* q = static_cast<const B*>(a.q) + q_at;
    if (a.q_wide) {
#pragma unroll
        for (int c = 0; c < N; c++) x[c] = *reinterpret_cast<const u32x4*>(q + (d + c * apart < a.dim ? d + c * apart : 0u));
    } else {
#pragma unroll
        for (int c = 0; c < N; c++) {
            B e[n];
#pragma unroll
            for (uint32_t i = 0; i < n; i++) e[i] = q[min(d + c * apart + i, a.dim - 1)];
#pragma unroll
            for (uint32_t i = 0; i < n; i++) if (d + c * apart + i >= a.dim) e[i] = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) x[c][i] = DT == kF32 ? (uint32_t)e[i * n / 4] : (uint32_t)e[i * n / 4] | (uint32_t)e[(i * n + n / 2) / 4] << 16;
        }
    }
    if (a.q_plain) return;
    const uint32_t sign = !a.negative ? 0u : DT == kF32 ? 0x80000000u : 0x80008000u;
#pragma unroll
    for (int c = 0; c < N; c++) {
        const bool in = !a.nothing && (!a.q_wide || d + c * apart < a.dim);
#pragma unroll
        for (int i = 0; i < 4; i++) x[c][i] = in ? x[c][i] ^ sign : 0u;
    }
}

// Weights are 2^kLift of themselves: f16 loses bits below 2^-14, and many small weights beside a large one would all lose the same ones.
template <int DT> constexpr float kLift = DT == kF16 ? 6.0f : 0.0f;

// One packed row over positions begin .. end - 1, by one wave and value by value: what takes the place of the matrix instructions where a
// result is not a number.  There a position that a row does not see has the weight 0, and 0 times an infinity or NaN that stands in it
// is NaN; here it is left out.  A wave takes all its rows so, whose positions
// follow each other through the table, the key and the sum over lanes: one NaN among the values that all rows of a sequence see makes 64 tokens at 4096 to 16384 1610 us
// instead of 430, 512 rows at position 16000 85 ms instead of 0.16.  Every lane gets the maximum (in powers of two) and the sum; sums[c] is of column lane + 64 c.
template <int DT, int D>
__device__ __forceinline__ void slow_row(const PagedArgs& a, int sequence, uint64_t q_at, uint32_t g, uint32_t begin, uint32_t end, uint32_t lane,
                                                   float& m, float& l, float (&sums)[(D + 63) / 64]) {
    typedef element_t<DT> B;
    constexpr int N = (D + 63) / 64;
    float q[N];
    m = -INFINITY; l = 0.0f;
#pragma unroll
    for (int c = 0; c < N; c++) {
        const uint32_t d = lane + 64 * c;
        q[c] = d < a.dim ? element_value<DT>(static_cast<const B*>(a.q)[q_at + d]) : 0.0f;
        sums[c] = 0.0f;
    }
    const uint32_t* row = a.plan.table + (size_t)sequence * a.plan.table_ld;
    for (uint32_t p = begin; p < end; p++) {
        const uint32_t b = p >> a.plan.shift, pg = b < a.plan.table_ld ? row[b] : 0xFFFFFFFFu;
        if (pg >= a.plan.pages) continue;
        const size_t at = (((((size_t)pg * a.kv_heads + g) << a.plan.shift) + (p & ((1u << a.plan.shift) - 1))) * D);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < N; c++) if (lane + 64 * c < a.dim) s = __builtin_fmaf(q[c], element_value<DT>(static_cast<const B*>(a.keys)[at + lane + 64 * c]), s);
        s = lh_group_sum(s, 64) * (a.nothing ? 0.0f : a.negative ? -a.scale2 : a.scale2);
        const float nm = fmaxf(m, s), base = nm == -INFINITY ? 0.0f : nm, f = exp2f(m - base), w = exp2f(s - base);
        l = l * f + w;
#pragma unroll
        for (int c = 0; c < N; c++) {
            const uint32_t d = lane + 64 * c;
            if (d < a.dim) sums[c] = __builtin_fmaf(w, element_value<DT>(static_cast<const B*>(a.values)[at + d]), sums[c] * f);
        }
        m = nm;
    }
}

// A workgroup per tile, kv head and split; its four waves take the split's positions in turn, each a quarter of them side by side,
// straight from global memory; their results meet in LDS.
//   S^T = K Q^T    a lane has packed row lane & 15 and positions 4 (lane / 16) .. + 3 of both halves of a step
//   O^T = V^T P^T  the weights are operands where they are; of V a lane loads D / 16 neighbouring columns of its eight positions, and
//                  pairs of positions are put together in registers, a column per product: no LDS on the way
// Weights of 16 bits are two terms, what the first leaves being the second: the products are few beside the loads, and what a result is off
// stays that of its own rounding.
// Memory binds it: 64 tokens over 4096 to 16384 positions of 8 kv heads of 128 (2.6 GB in pages of 16 positions, runs of 4 KB) 421 us, 6.2 TB/s,
// where reading alone reaches 6.2 to 6.8 in runs of 8 KB; 15 % of a SIMD's time is vector and matrix work.  One token over 32768 (134 MB) 24 us.
// 256 columns of 16 bits take 256 registers and keep two values in scratch (12 bytes a lane); f32 of 192 and 256 takes 272 and 324, one wave a SIMD.
// The next step's keys are requested when this one's are used, its values likewise (the 64 tokens 450 -> 444 us).
// The hint that nothing is read again, for caches that would push everything else out from near the chip: 472 -> 450, the token with its pages in memory
// 31.9 -> 28.9 (where the last launch has left them near, 26.9 -> 27.3).  Pages that sequences share are read again, and soon: 64 tokens over the same 16384
// positions take 535 with the hint and 301 without.  So a wave looks whether the sequence before or behind its own begins with the same page here.  Nor
// where a lane's part of a value is not 16 bytes: two pieces then touch each line twice (16 tokens of 256 columns 45 without, 51 with it).
template <int DT, int D>
__global__ __launch_bounds__(256, DT == kF32 ? (D <= 128 ? 2 : 1) : D <= 128 ? 3 : 2) void paged_rows_kernel(const PagedArgs a) {
    typedef element_t<DT> B;
    constexpr bool WIDE = DT == kF32, AHEAD = !WIDE || D <= 64;      // (wider rows of 32 bits leave no registers for it)
    constexpr int DL = D / 16, kRow = D + 4, KC = WIDE ? D / 16 : D / 32, VW = WIDE ? DL : DL / 2;
    constexpr bool HINT = VW == 4;
    extern __shared__ __align__(16) float slab[];             // [4 waves][16][kRow]
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), gr = lane >> 4, lr = lane & 15;
    const uint32_t n = a.by_heads.of(blockIdx.x), g = blockIdx.x - n * a.kv_heads;
    const Tile tile = tile_of<16, 32, false>(a, n, lane);
    if (tile.sequence < 0) return;
    const uint32_t R = a.group.d, packed = tile.row0 + min(lr, tile.count - 1), row = a.group.of(packed), head = g * R + packed - row * R;
    const bool on = lr < tile.count;
    const uint32_t last_row = a.group.of(tile.row0 + tile.count - 1), first_row = a.group.of(tile.row0);
    const Seen mine = seen_by(a, tile, row), first_seen = seen_by(a, tile, first_row), last_seen = seen_by(a, tile, last_row);
    const Part part = part_of<32>(tile, first_seen.lo, last_seen.hi, tile.split);
    if (tile.split >= part.used) return;
    const uint32_t per = (part.end - part.begin + 3) / 4, begin = min(part.begin + wave * per, part.end), end = min(begin + per, part.end);
    const uint64_t q_at = (uint64_t)(tile.first + row) * a.q_ld + (uint64_t)head * a.dim;

    // (the table is asked first: the queries are many small pieces, and its way begins behind theirs otherwise)
    Pages pages{a.plan.table + (size_t)tile.sequence * a.plan.table_ld, (last_seen.hi + (1u << a.plan.shift) - 1) >> a.plan.shift, 0, 0, 0};
    bool stream = false;
    uint32_t beside = ~0u;
    if (begin < end) {
        const uint32_t block = (begin * 32) >> a.plan.shift, s = tile.sequence + (lane & 1) * 2 - 1;
        pages.ask(a.plan, block, lane);
        if (HINT && a.stream && lane < 2 && s < a.plan.sequences && block < a.plan.table_ld) beside = a.plan.table[(size_t)s * a.plan.table_ld + block];
    }
    u32x4 qf[KC];
    load_query<DT>(a, q_at, gr * (WIDE ? 4 : 8), WIDE ? 16 : 32, qf);
    pages.settle(a.plan, lane);
    if (HINT && a.stream) stream = !__ballot(lane < 2 && beside == (uint32_t)__builtin_amdgcn_readfirstlane(pages.entry));
    const float scale2 = a.scale2;
    float m = -INFINITY, l = 0.0f;
    lh_f32x4 o[DL];
#pragma unroll
    for (int i = 0; i < DL; i++) o[i] = (lh_f32x4){0.f, 0.f, 0.f, 0.f};

    const uint32_t in_page = (1u << a.plan.shift) - 1;
    // Where step b's halves stand: the page's rows for this kv head, from the half's first slot on.
    uint64_t base[2];
    bool next_there[2];
    auto locate = [&](uint32_t b) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t p = b * 32 + 16 * h, block = p >> a.plan.shift;
            pages.reach(a.plan, block, lane);
            next_there[h] = pages.has(block);
            base[h] = (((((uint64_t)pages.of(a.plan, block) * a.kv_heads + g) << a.plan.shift) + (p & in_page))) * D;
        }
    };
    u32x4 kf[2][KC];
    uint32_t v[2][4][VW];
    auto keys_of = [&](auto hint) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const B* K = static_cast<const B*>(a.keys) + base[h] + lr * D + gr * (WIDE ? 4 : 8);
#pragma unroll
            for (int c = 0; c < KC; c++) kf[h][c] = load16<hint()>(K + c * (WIDE ? 16 : 32));
        }
    };
    auto values_of = [&](auto hint) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const B* V = static_cast<const B*>(a.values) + base[h] + gr * 4 * D + lr * DL;
#pragma unroll
            for (int j = 0; j < 4; j++) load_words<hint()>(V + j * D, v[h][j]);
        }
    };
    // (both ways are the same loads but for the hint, and the compiler would make one without it of them)
    auto by_hint = [&](auto&& load) __attribute__((always_inline)) {
        if constexpr (HINT) if (stream) {
            asm volatile("" ::: "memory");
            load(std::true_type{});
            asm volatile("" ::: "memory");
            return;
        }
        load(std::false_type{});
    };
    auto load_keys = [&]() __attribute__((always_inline)) { by_hint(keys_of); };
    auto load_values = [&]() __attribute__((always_inline)) { by_hint(values_of); };
    if (AHEAD && begin < end) { locate(begin); load_keys(); load_values(); }
    for (uint32_t b = begin; b < end; b++) {
        if (!AHEAD) { locate(b); load_keys(); load_values(); }
        const bool there[2] = {next_there[0], next_there[1]};
        lh_f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = (lh_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; c++) {
                if constexpr (WIDE) {
                    const lh_f32x4 x = __builtin_bit_cast(lh_f32x4, kf[h][c]), y = __builtin_bit_cast(lh_f32x4, qf[c]);
#pragma unroll
                    for (int j = 0; j < 4; j++) s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], s[h], 0, 0, 0);
                } else {
                    s[h] = product<DT>(kf[h][c], qf[c], s[h]);
                }
            }
        }
        if (AHEAD && b + 1 < end) { locate(b + 1); load_keys(); }
        float p[8], mx = -INFINITY;
        const bool whole = b * 32 >= last_seen.lo && b * 32 + 32 <= first_seen.hi && there[0] && there[1];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = s[i >> 2][i & 3] * scale2;
            if (!whole) {
                const uint32_t at = b * 32 + (i >> 2) * 16 + gr * 4 + (i & 3);
                if (at < mine.lo || at >= mine.hi || !there[i >> 2]) p[i] = -INFINITY;
                if (at >= last_seen.hi || at < first_seen.lo || !there[i >> 2]) {      // seen by none: may be anything
#pragma unroll
                    for (int e = 0; e < VW; e++) v[i >> 2][i & 3][e] = 0;
                }
            }
            mx = fmaxf(mx, p[i]);
        }
        const float nm = fmaxf(m, lh_column_max(mx)), base_m = nm == -INFINITY ? 0.0f : nm, alpha = __builtin_amdgcn_exp2f(m - base_m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) { p[i] = __builtin_amdgcn_exp2f(p[i] - (base_m - kLift<DT>)); sum += p[i]; }
        l = l * alpha + sum;                                  // this lane's positions; the four lanes of a row are added at the end
        m = nm;
#pragma unroll
        for (int i = 0; i < DL; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] *= alpha;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < DL; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, v[j >> 2][j & 3][i]), p[j], o[i], 0, 0, 0);
        } else {
            u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                hi[i] = pack2<DT>(p[2 * i], p[2 * i + 1]);
                lo[i] = pack2<DT>(p[2 * i] - low<DT>(hi[i]), p[2 * i + 1] - high<DT>(hi[i]));
            }
#pragma unroll
            for (int i = 0; i < DL; i++) {
                const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
                u32x4 x;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __builtin_amdgcn_perm(v[e >> 1][(e & 1) * 2 + 1][i / 2], v[e >> 1][(e & 1) * 2][i / 2], sel);
                o[i] = product<DT>(x, hi, o[i]);
                o[i] = product<DT>(x, lo, o[i]);
            }
        }
        if (AHEAD && b + 1 < end) load_values();
    }
    // The wave's results: row lr, columns (4 gr + j) DL + i.
    float* own = slab + wave * 16 * kRow;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < DL; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) odd = odd || o[i][j] != o[i][j];
    l = lh_column_sum(l);
    if (__any(on && odd)) {
        for (uint32_t r = 0; r < tile.count; r++) {
            const uint32_t pk = tile.row0 + r, rw = a.group.of(pk);
            const Seen sn = seen_by(a, tile, rw);
            float sm, sl, sums[(D + 63) / 64];
            slow_row<DT, D>(a, tile.sequence, (uint64_t)(tile.first + rw) * a.q_ld + (uint64_t)(g * R + pk - rw * R) * a.dim, g, max(begin * 32, sn.lo), min(end * 32, sn.hi), lane, sm, sl, sums);
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; c++) if (lane + 64 * c < D) own[r * kRow + lane + 64 * c] = sums[c];
            if (lane == 0) { own[r * kRow + D] = sm; own[r * kRow + D + 1] = sl; }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float* to = own + lr * kRow + (4 * gr + j) * DL;
            if constexpr (DL % 4 == 0) {
#pragma unroll
                for (int i = 0; i < DL; i += 4) *reinterpret_cast<lh_f32x4*>(to + i) = (lh_f32x4){o[i][j], o[i + 1][j], o[i + 2][j], o[i + 3][j]};
            } else {
#pragma unroll
                for (int i = 0; i < DL; i++) to[i] = o[i][j];
            }
        }
        if (gr == 0) { own[lr * kRow + D] = m - kLift<DT>; own[lr * kRow + D + 1] = l; }
    }
    __syncthreads();
    const uint32_t r = tid >> 4, c0 = (tid & 15) * 4;
    if (r >= tile.count) return;
    float top = -INFINITY, total = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, slab[(w * 16 + r) * kRow + D]);
    const uint32_t pk = tile.row0 + r, rw = a.group.of(pk), hd = g * R + pk - rw * R;
    const bool alone = part.used == 1;
    const float sink = alone && a.sink ? a.sink[hd] * kLog2e : -INFINITY, ref = fmaxf(top, sink), zero = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        f[w] = __builtin_amdgcn_exp2f(slab[(w * 16 + r) * kRow + D] - zero);
        total += f[w] * slab[(w * 16 + r) * kRow + D + 1];
    }
    const float all = total + __builtin_amdgcn_exp2f(sink - zero), inv = alone ? (total == 0.0f ? 0.0f : 1.0f / all) : 1.0f;
    float* rec = alone ? nullptr : a.partial + ((tile.record_of(a, g) + tile.split) * a.rows_kept + r) * kRow;
    if (rec && c0 == 0) { rec[D] = zero; rec[D + 1] = total; }
    B* out = static_cast<B*>(a.out) + (uint64_t)(tile.first + rw) * a.out_ld + (uint64_t)hd * a.dim;
    for (uint32_t c = c0; c < D; c += 64) {
        lh_f32x4 x = (lh_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const lh_f32x4 y = *reinterpret_cast<const lh_f32x4*>(slab + (w * 16 + r) * kRow + c);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] += f[w] * y[j];      // (a NaN that weighs nothing is one all the same; a wave that saw nothing has zeros)
        }
        if (rec) { *reinterpret_cast<lh_f32x4*>(rec + c) = x; continue; }
#pragma unroll
        for (int j = 0; j < 4; j++) if (c + j < a.dim) out[c + j] = element_bits<DT>(x[j] * inv);
    }
}

typedef float lh_f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

// 16 bytes a lane from base + from straight to LDS, lane by lane from byte `to` on (the same in all lanes).  No registers are written, so
// nothing can be read too early but LDS itself, behind wait_for_loads and a barrier.  (With the builtin for it the compiler has every
// transposing read wait for all such loads, the next step's among them.  m0 is the compiler's own and holds nothing over an instruction.)
__device__ __forceinline__ void load_to_lds(uint32_t to, const void* base, uint32_t from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(from), "s"(base) : "memory");
}
// (The builtin tells the compiler, too, that its own loads are there: else it would wait for them, and with them for these, at their first use.)
__device__ __forceinline__ void wait_for_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); asm volatile("" ::: "memory"); }

template <int DT>
__device__ __forceinline__ lh_f32x16 product(u32x4 x, u32x4 y, lh_f32x16 c) {
    if constexpr (DT == kF16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lh_f16x8, x), __builtin_bit_cast(lh_f16x8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lh_bf16x8, x), __builtin_bit_cast(lh_bf16x8, y), c, 0, 0, 0);
}

// A lane's columns c + 4 half .. + 3 and c + 8 + 4 half .. + 3 of its row, stored 16 bytes at a time: the lower half of the wave takes c .. c + 7
// of its rows, the upper half the rest.  All lanes call it.
template <int DT>
__device__ __forceinline__ void store_pair(element_t<DT>* out, uint32_t c, uint32_t half, lh_f32x4 x, lh_f32x4 y, bool on, uint32_t dim, uint32_t wide) {
    const uint32_t x0 = pack2<DT>(x[0], x[1]), x1 = pack2<DT>(x[2], x[3]), y0 = pack2<DT>(y[0], y[1]), y1 = pack2<DT>(y[2], y[3]);
    const auto p = __builtin_amdgcn_permlane32_swap(x0, y0, false, false), q = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
    const u32x4 w = {p[0], q[0], p[1], q[1]};
    c += 8 * half;
    if (!on) return;
    if (wide) {
        if (c < dim) *reinterpret_cast<u32x4*>(out + c) = w;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) if (c + j < dim) out[c + j] = (element_t<DT>)(w[j / 2] >> 16 * (j & 1));
    }
}

// A key row's pieces are at c ^ key_place(row): rows of 16 pieces fill the banks, shorter ones do so together.
template <uint32_t PIECES>
__device__ __forceinline__ constexpr uint32_t key_place(uint32_t row) { return PIECES % 16 == 0 ? row & 15 : PIECES % 8 == 0 ? (row >> 1) & 7 : (row >> 2) & 3; }

// Many rows, 16-bit types: a workgroup per tile of 128 packed rows, kv head and split.  Each of its four waves has 32 rows, all of them
// share the steps of KT positions, whose keys and values go from memory to LDS without registers, the next step's while this one is used.
//   S^T = K Q^T    32 x 32 x 16: a lane has packed row lane & 31 and half of the positions, so maximum and sum are its own registers'
//   O^T = V^T P^T  the weights are operands where they are; V, in LDS as it is in memory, is read by the transposing ds_read_b64_tr_b16
// A weight is rounded once to 16 bits, which is what a result is off beside its own rounding: in bf16 0.0023 of it where that alone makes 0.0017.
// (A second term as for few rows would be half as many products again.)
// Issue binds it most: 512 rows at position 16000 of 32 heads over 8 kv heads of 128 take 136 to 141 us (from card to card), 0.97 to 1.0 PFLOP/s, at the 2.0 GHz that
// the chip keeps there; the matrix instructions fill 46 % of a SIMD's time and the vector ones, which add to it, another 30.  The rest, 24 %, is waits: a step's barrier
// and its loads, and reads of LDS, which is busy for 23 % of the time (every wave reads all keys and values of a step for its 32 rows; no bank conflicts).  Four prompts of
// 2048 to 4096 rows of 16 heads over 4: 206 to 221 us, 0.85 to 0.91.  The wave's priority is raised for the products (prompts 233 -> 231), operands are a group ahead
// (chunk 157 -> 153.5), the buffers' places are constants of a loop of two steps (156 -> 153.5).  256 columns: a wave a SIMD, 2000 rows of 8 heads
// over one 62 us, 0.53.
// In LDS the 16-byte pieces of a row change places by the row's low bits, so that neither read meets itself in one of the 64 banks: of
// 16 neighbouring key rows the same piece is in 16 places (key_place), of four value rows the same four pieces in four.
template <int DT, int D>
__global__ __launch_bounds__(256, D <= 192 ? 2 : 1) void paged_tiles_kernel(const PagedArgs a) {
    typedef element_t<DT> B;
    constexpr uint32_t KT = tile_step(D), SUB = KT / 32, KC = D / 16, TD = D / 32, CR = D / 8, PART = KT / 4, LOADS = PART * D / 512, kRow = D + 4;
    constexpr uint32_t VSWAP = CR % 16 == 0 ? 3 : CR % 8 == 0 ? 1 : 0;
    constexpr bool AHEAD = D != 192;                          // (which leaves no registers for it; 256 have all of a SIMD's for one wave)
    extern __shared__ __align__(16) uint16_t stage_memory[];
    lds_u16* const stage = (lds_u16*)stage_memory;            // [2][keys, values][KT][D]
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, lr = lane & 31;
    const uint32_t n = a.by_heads.of(blockIdx.x), g = blockIdx.x - n * a.kv_heads;
    const Tile tile = tile_of<128, KT, false>(a, a.parts - 1 - n, lane);      // a sequence's last rows, which see most, first
    if (tile.sequence < 0) return;
    const uint32_t R = a.group.d, last_row = a.group.of(tile.row0 + tile.count - 1);
    const Seen first_seen = seen_by(a, tile, a.group.of(tile.row0)), last_seen = seen_by(a, tile, last_row);
    const Part part = part_of<KT>(tile, first_seen.lo, last_seen.hi, tile.split);
    if (tile.split >= part.used) return;
    // the wave's rows
    const bool busy = wave * 32 < tile.count;
    const uint32_t in_tile = min(wave * 32 + lr, tile.count - 1), packed = tile.row0 + in_tile, row = a.group.of(packed), head = g * R + packed - row * R;
    const bool on = wave * 32 + lr < tile.count;
    const Seen mine = seen_by(a, tile, row), wave_first = seen_by(a, tile, min(a.group.of(tile.row0 + wave * 32), last_row)),
               wave_last = seen_by(a, tile, a.group.of(tile.row0 + min(wave * 32 + 31, tile.count - 1)));
    const uint64_t q_at = (uint64_t)(tile.first + row) * a.q_ld + (uint64_t)head * a.dim;
    u32x4 qf[KC];
    load_query<DT>(a, q_at, half * 8, 16, qf);

    // where a lane's pieces come from, in bytes from the part's first row on
    uint32_t kfrom[LOADS], vfrom[LOADS];
#pragma unroll
    for (uint32_t j = 0; j < LOADS; j++) {
        const uint32_t id = j * 64 + lane, r = id / CR, c = id % CR;
        kfrom[j] = (r * D + (c ^ key_place<CR>(wave * PART + r)) * 8) * 2;
        vfrom[j] = (r * D + (c ^ (((wave * PART + r) & VSWAP) << 2)) * 8) * 2;
    }
    Pages pages{a.plan.table + (size_t)tile.sequence * a.plan.table_ld, (last_seen.hi + (1u << a.plan.shift) - 1) >> a.plan.shift, 0, 0, 0};
    const uint32_t in_page = (1u << a.plan.shift) - 1;
    if (part.begin < part.end) pages.load(a.plan, (part.begin * KT) >> a.plan.shift, lane);
    // Requests step b into buffer `at`; returns which quarters of it are there.
    auto request = [&](uint32_t b, uint32_t at) __attribute__((always_inline)) {
        const uint32_t block = (b * KT + wave * PART) >> a.plan.shift, first = (b * KT) >> a.plan.shift;
        if (first - pages.held > 60) pages.load(a.plan, first, lane);             // (a step has four at most)
        uint32_t there = 15;
        if (pages.there != ~0ull) {
            there = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) there |= (uint32_t)pages.has((b * KT + i * PART) >> a.plan.shift) << i;
        }
        const uint64_t base = ((((uint64_t)pages.of(a.plan, block) * a.kv_heads + g) << a.plan.shift) + ((b * KT + wave * PART) & in_page)) * D;
        const B *K = static_cast<const B*>(a.keys) + base, *V = static_cast<const B*>(a.values) + base;
        const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(stage + (at * 2 * KT + wave * PART) * D));
#pragma unroll
        for (uint32_t j = 0; j < LOADS; j++) load_to_lds(to + j * 1024, K, kfrom[j]);
#pragma unroll
        for (uint32_t j = 0; j < LOADS; j++) load_to_lds(to + KT * D * 2 + j * 1024, V, vfrom[j]);
        return there;
    };
    // where a lane reads operands, in values: of keys row lr, of values row 4 half + (lane & 15) / 4
    constexpr uint32_t KO = CR % 16 == 0 ? 8 : CR % 8 == 0 ? 4 : 2, VO = VSWAP == 3 ? 4 : VSWAP == 1 ? 2 : 1;
    uint32_t kat[KO], vat[VO];
#pragma unroll
    for (uint32_t c = 0; c < KO; c++) kat[c] = lr * D + ((c * 2 + half) ^ key_place<CR>(lr)) * 8;
#pragma unroll
    for (uint32_t c = 0; c < VO; c++) {
        const uint32_t i = lane & 15, r = 4 * half + (i >> 2), piece = c * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
        vat[c] = r * D + (piece ^ ((r & VSWAP) << 2)) * 8 + (i & 1) * 4;
    }

    const float scale2 = a.scale2;
    float m = -INFINITY, l = 0.0f;
    lh_f32x16 o[TD];
#pragma unroll
    for (uint32_t d = 0; d < TD; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    wait_for_loads();                                         // queries and table, so that the compiler waits for neither later
    uint32_t next_there = part.begin < part.end ? request(part.begin, 0) : 0u;
    auto step = [&](uint32_t b, auto buffer) __attribute__((always_inline)) {
        constexpr uint32_t at = decltype(buffer)::value;      // a constant: it goes into the reads' offsets
        const uint32_t there = next_there, p0 = b * KT;
        wait_for_loads();
        __syncthreads();                                      // the step is there, and nobody reads the other buffer any more
        if (b + 1 < part.end) next_there = request(b + 1, at ^ 1);
        const lds_u16 *K = stage + at * 2 * KT * D, *V = K + KT * D;
        if (p0 + KT > last_seen.hi || p0 < first_seen.lo || there != 15u) {      // positions that no row sees: what stands there may be anything
            lds_u16* v = stage + (at * 2 + 1) * KT * D;
            for (uint32_t i = tid; i < KT * CR; i += 256) {
                const uint32_t r = i / CR, p = p0 + r;
                if (p >= last_seen.hi || p < first_seen.lo || !(there >> (r / PART) & 1)) *(lds_u32x4*)(v + i * 8) = (u32x4){0, 0, 0, 0};
            }
            lh_lds_barrier();
        }
        if (!busy || p0 >= wave_last.hi || p0 + KT <= wave_first.lo) return;
        // AHEAD: operands are requested a group of products ahead: 32 positions of keys, 32 columns of values
        lh_f32x16 s[SUB];
        u32x4 kf[2][KC], vf[2][2 * SUB];
        auto keys_of = [&](uint32_t u, u32x4 (&x)[KC]) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t c = 0; c < KC; c++) x[c] = *(const lds_u32x4*)(K + kat[c % KO] + u * 32 * D + c / KO * KO * 16);
        };
        auto values_of = [&](uint32_t d, u32x4 (&x)[2 * SUB]) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t k = 0; k < 2 * SUB; k++) {
                const lds_u16* v = V + vat[d % VO] + k * 16 * D + d / VO * VO * 32;
                const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)v));
                const uint2 z = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v + 8 * D)));
                x[k] = (u32x4){y.x, y.y, z.x, z.y};
            }
        };
        if (AHEAD) keys_of(0, kf[0]);
#pragma unroll
        for (uint32_t u = 0; u < SUB; u++) {
            if (!AHEAD) keys_of(u, kf[u & 1]);
            else if (u + 1 < SUB) keys_of(u + 1, kf[(u + 1) & 1]);
            else values_of(0, vf[0]);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 16; i++) s[u][i] = 0.0f;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (uint32_t c = 0; c < KC; c++) s[u] = product<DT>(kf[u & 1][c], qf[c], s[u]);
            __builtin_amdgcn_s_setprio(0);
        }
        const bool whole = p0 >= wave_last.lo && p0 + KT <= wave_first.hi && there == 15u;
        if (!whole)
#pragma unroll
            for (uint32_t u = 0; u < SUB; u++)
#pragma unroll
                for (uint32_t i = 0; i < 16; i++) {
                    const uint32_t r = u * 32 + 8 * (i / 4) + 4 * half + (i & 3), p = p0 + r;
                    if (p < mine.lo || p >= mine.hi || !(there >> (r / PART) & 1)) s[u][i] = -INFINITY;
                }
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t u = 0; u < SUB; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[u][i]);
        float ma, mb;
        lh_pair32(mx, ma, mb);
        const float nm = fmaxf(m, fmaxf(ma, mb) * scale2 - kLift<DT>);
        // The reference of the weights follows the maximum only where that has grown 2^8 times: until then they are at most 2^8 (f16: 2^14), which
        // all types hold as exactly as 1.
        if (__any(nm > m + 8.0f)) {
            const float alpha = __builtin_amdgcn_exp2f(m - (nm == -INFINITY ? 0.0f : nm));
            l *= alpha;
            m = nm;
#pragma unroll
            for (uint32_t d = 0; d < TD; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= alpha;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        u32x4 w[2 * SUB];
        float sum = 0.0f;
#pragma unroll
        for (uint32_t u = 0; u < SUB; u++)
#pragma unroll
            for (uint32_t i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], scale2, -base)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i + 1], scale2, -base));
                sum += x + y;
                w[2 * u + i / 8][i / 2 % 4] = pack2<DT>(x, y);
            }
        l += sum;
#pragma unroll
        for (uint32_t d = 0; d < TD; d++) {
            if (d == 0) __builtin_amdgcn_s_setprio(1);
            if (!AHEAD) values_of(d, vf[d & 1]);
            else if (d + 1 < TD) values_of(d + 1, vf[(d + 1) & 1]);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t k = 0; k < 2 * SUB; k++) o[d] = product<DT>(vf[d & 1][k], w[k], o[d]);
            if (d + 1 == TD) __builtin_amdgcn_s_setprio(0);
        }
    };
    for (uint32_t b = part.begin; b < part.end; b += 2) {
        step(b, std::integral_constant<uint32_t, 0>());
        if (b + 1 < part.end) step(b + 1, std::integral_constant<uint32_t, 1>());
    }
    if (!busy) return;
    const bool alone = part.used == 1;
    // a record is in the order in which the waves have it: [wave][16-byte piece][lane], and maximum and sum of the 128 rows
    float* rec = alone ? nullptr : a.partial + (tile.record_of(a, g) + tile.split) * 128 * kRow;
    float2* stats = reinterpret_cast<float2*>(rec + 128 * D) + wave * 32;
    rec += wave * 32 * D;
    bool odd = false;
#pragma unroll
    for (uint32_t d = 0; d < TD; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) odd = odd || !(fabsf(o[d][i]) < INFINITY);      // (weights above 1 may have made the infinity)
    if (__any(on && odd)) {
        for (uint32_t r = 0; r < 32 && wave * 32 + r < tile.count; r++) {
            const uint32_t pk = tile.row0 + wave * 32 + r, rw = a.group.of(pk), hd = g * R + pk - rw * R;
            const Seen sn = seen_by(a, tile, rw);
            float sm, sl, sums[(D + 63) / 64];
            slow_row<DT, D>(a, tile.sequence, (uint64_t)(tile.first + rw) * a.q_ld + (uint64_t)hd * a.dim, g, max(part.begin * KT, sn.lo), min(part.end * KT, sn.hi), lane, sm, sl, sums);
            const float ref = alone && a.sink ? fmaxf(sm, a.sink[hd] * kLog2e) : sm, zero = ref == -INFINITY ? 0.0f : ref, f = __builtin_amdgcn_exp2f(sm - zero);
            const float total = sl * f + (alone && a.sink ? __builtin_amdgcn_exp2f(a.sink[hd] * kLog2e - zero) : 0.0f), scale = alone ? (sl == 0.0f ? 0.0f : f / total) : 1.0f;
            if (!alone && lane == 0) stats[r] = make_float2(sm == -INFINITY ? 0.0f : sm, sl);
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; c++) {
                const uint32_t d = lane + 64 * c;
                if (!alone) { if (d < D) rec[(d / 8 * 64 + d / 4 % 2 * 32 + r) * 4 + d % 4] = sums[c]; }
                else if (d < a.dim) static_cast<B*>(a.out)[(uint64_t)(tile.first + rw) * a.out_ld + (uint64_t)hd * a.dim + d] = element_bits<DT>(sums[c] * scale);
            }
        }
        return;
    }
    l = lh_sum32_f(l);
    // a lane has columns 32 d + 8 i + 4 half .. + 3 of its row
    if (!alone) {
#pragma unroll
        for (uint32_t d = 0; d < TD; d++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                *reinterpret_cast<lh_f32x4*>(rec + ((4 * d + i) * 64 + lane) * 4) = (lh_f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (half == 0) stats[lr] = make_float2(m == -INFINITY ? 0.0f : m, l);
        return;
    }
    const float sink = a.sink ? a.sink[head] * kLog2e : -INFINITY, ref = fmaxf(m, sink), zero = ref == -INFINITY ? 0.0f : ref, f = __builtin_amdgcn_exp2f(m - zero);
    const float inv = l == 0.0f ? 0.0f : f / (l * f + __builtin_amdgcn_exp2f(sink - zero));
    B* out = static_cast<B*>(a.out) + (uint64_t)(tile.first + row) * a.out_ld + (uint64_t)head * a.dim;
#pragma unroll
    for (uint32_t d = 0; d < TD; d++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i += 2) {
            lh_f32x4 x, y;
#pragma unroll
            for (int j = 0; j < 4; j++) { x[j] = o[d][4 * i + j] * inv; y[j] = o[d][4 * i + 4 + j] * inv; }
            store_pair<DT>(out, 32 * d + 8 * i, half, x, y, on, a.dim, a.out_wide);
        }
}

// The splits of a tile of 128 rows, in the order in which the waves' registers had them, so that loads and stores are whole lines (512 rows of 32 heads in four parts:
// 10 us from rows, 8 so, and the kernel before it 3 less): a lane has two 16-byte pieces of a record, four splits on their way at a time.  MANY (more than four
// splits): a workgroup's four waves take the splits of the same pieces in turn and meet in LDS.
template <int DT, int D, bool MANY>
__global__ __launch_bounds__(256) void paged_merge_tiles_kernel(const PagedArgs a) {
    typedef element_t<DT> B;
    constexpr uint32_t kRow = D + 4, KT = tile_step(D), PAIRS = D / 16, WGS = MANY ? 4 * PAIRS : PAIRS, BATCH = 4;
    __shared__ lh_f32x4 sums[MANY ? 4 : 1][2][64];
    __shared__ float2 totals[MANY ? 4 : 1][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63, half = lane >> 5, me = tid >> 6;
    const uint32_t tg = blockIdx.x / WGS, t = a.by_heads.of(tg), g = tg - t * a.kv_heads, unit = MANY ? blockIdx.x % WGS : blockIdx.x % WGS * 4 + me;
    const Tile tile = tile_of<128, KT, true>(a, t, lane);
    const uint32_t wave = unit / PAIRS, piece = unit % PAIRS * 2;      // of the wave that wrote them
    if (tile.sequence < 0 || wave * 32 >= tile.count) return;
    const uint32_t R = a.group.d;
    const Part part = part_of<KT>(tile, seen_by(a, tile, a.group.of(tile.row0)).lo, seen_by(a, tile, a.group.of(tile.row0 + tile.count - 1)).hi, 0);
    if (part.used == 1) return;
    const bool on = wave * 32 + (lane & 31) < tile.count;
    const uint32_t r = min(wave * 32 + (lane & 31), tile.count - 1), pk = tile.row0 + r, rw = a.group.of(pk), hd = g * R + pk - rw * R;
    const float* rec = a.partial + tile.record_of(a, g) * 128 * kRow;
    const size_t stride = 128 * kRow;
    const float sink = a.sink ? a.sink[hd] * kLog2e : -INFINITY;
    lh_f32x4 x = (lh_f32x4){0.f, 0.f, 0.f, 0.f}, y = x;
    float m = -INFINITY, l = 0.0f;
    // sums p, q of weight .y with maximum .x join x, y
    auto join = [&](auto& st, auto& p, auto& q, auto count) __attribute__((always_inline)) {
        constexpr uint32_t n = decltype(count)::value;
        float nm = m;
#pragma unroll
        for (uint32_t i = 0; i < n; i++) {
            if (st[i].y == 0.0f) st[i].x = -INFINITY;          // nothing that weighs anything: zeros, or a NaN that was seen
            nm = fmaxf(nm, st[i].x);
        }
        const float zero = nm == -INFINITY ? 0.0f : nm, before = __builtin_amdgcn_exp2f(m - zero);
        m = nm;
        l *= before;
#pragma unroll
        for (int j = 0; j < 4; j++) { x[j] *= before; y[j] *= before; }
#pragma unroll
        for (uint32_t i = 0; i < n; i++) {
            const float f = __builtin_amdgcn_exp2f(st[i].x - zero);
            l += f * st[i].y;
#pragma unroll
            for (int j = 0; j < 4; j++) { x[j] += f * p[i][j]; y[j] += f * q[i][j]; }
        }
    };
    constexpr uint32_t each = MANY ? 4 : 1;
    for (uint32_t s0 = MANY ? me : 0; s0 < part.used; s0 += each * BATCH) {
        lh_f32x4 p[BATCH], q[BATCH];
        float2 st[BATCH];
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) {
            const float* from = rec + min(s0 + i * each, part.used - 1) * stride;
            p[i] = *reinterpret_cast<const lh_f32x4*>(from + wave * 32 * D + (piece * 64 + lane) * 4);
            q[i] = *reinterpret_cast<const lh_f32x4*>(from + wave * 32 * D + (piece * 64 + 64 + lane) * 4);
            st[i] = reinterpret_cast<const float2*>(from + 128 * D)[r];
        }
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) if (s0 + i * each >= part.used) { st[i].y = 0.0f; p[i] = q[i] = (lh_f32x4){0.f, 0.f, 0.f, 0.f}; }
        join(st, p, q, std::integral_constant<uint32_t, BATCH>());
    }
    if constexpr (MANY) {
        sums[me][0][lane] = x; sums[me][1][lane] = y; totals[me][lane] = make_float2(m, l);
        __syncthreads();
        if (me) return;
        lh_f32x4 p[3], q[3];
        float2 st[3];
#pragma unroll
        for (uint32_t i = 0; i < 3; i++) { p[i] = sums[i + 1][0][lane]; q[i] = sums[i + 1][1][lane]; st[i] = totals[i + 1][lane]; }
        join(st, p, q, std::integral_constant<uint32_t, 3>());
    }
    const float ref = fmaxf(m, sink), zero = ref == -INFINITY ? 0.0f : ref, f = __builtin_amdgcn_exp2f(m - zero);
    const float inv = l == 0.0f ? 0.0f : f / (l * f + __builtin_amdgcn_exp2f(sink - zero));
#pragma unroll
    for (int j = 0; j < 4; j++) { x[j] *= inv; y[j] *= inv; }
    store_pair<DT>(static_cast<B*>(a.out) + (uint64_t)(tile.first + rw) * a.out_ld + (uint64_t)hd * a.dim, piece * 8, half, x, y, on, a.dim, a.out_wide);
}

// The splits of a tile of 16 rows: D / 4 lanes take a split's sums, four columns each, eight splits on their way at a time, and keep a
// running maximum of what they have seen.  FEW: these lanes are all that a row has.  Else a workgroup a row, whose
// groups of lanes take the splits in turn and meet in LDS.
template <int DT, int D, bool FEW>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedArgs a) {
    typedef element_t<DT> B;
    constexpr uint32_t ROWS = 16, STEP = 32, kRow = D + 4, QUADS = D / 4, GROUPS = 256 / QUADS, PER = FEW ? GROUPS : 1, BATCH = 8;
    __shared__ lh_f32x4 sums[FEW ? 1 : 256];
    __shared__ float2 totals[GROUPS];
    const uint32_t tid = threadIdx.x, lane = tid & 63, grp = tid / QUADS, c = tid % QUADS * 4;
    const uint32_t t = a.by_heads.of(blockIdx.x), g = blockIdx.x - t * a.kv_heads, r = blockIdx.y * PER + (FEW ? grp : 0);
    const Tile tile = tile_of<ROWS, STEP, true>(a, t, lane);
    if (tile.sequence < 0 || (FEW && grp >= GROUPS) || r >= tile.count) return;
    const uint32_t R = a.group.d, pk = tile.row0 + r, rw = a.group.of(pk), hd = g * R + pk - rw * R;
    const Part part = part_of<STEP>(tile, seen_by(a, tile, a.group.of(tile.row0)).lo, seen_by(a, tile, a.group.of(tile.row0 + tile.count - 1)).hi, 0);
    if (part.used == 1) return;
    const float* rec = a.partial + (tile.record_of(a, g) * a.rows_kept + r) * kRow;
    const size_t stride = (size_t)a.rows_kept * kRow;
    const float sink = a.sink ? a.sink[hd] * kLog2e : -INFINITY;
    lh_f32x4 x = (lh_f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    const uint32_t each = FEW ? 1 : GROUPS;
    for (uint32_t s0 = FEW ? 0 : grp; s0 < part.used && grp < GROUPS; s0 += each * BATCH) {
        lh_f32x4 y[BATCH];
        float2 st[BATCH];
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) {
            const float* p = rec + min(s0 + i * each, part.used - 1) * stride;
            y[i] = *reinterpret_cast<const lh_f32x4*>(p + c);
            st[i] = *reinterpret_cast<const float2*>(p + D);
        }
        float nm = m;
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) {
            if (s0 + i * each >= part.used) { st[i].y = 0.0f; y[i] = (lh_f32x4){0.f, 0.f, 0.f, 0.f}; }
            if (st[i].y == 0.0f) st[i].x = -INFINITY;          // nothing that weighs anything: zeros, or a NaN that was seen
            nm = fmaxf(nm, st[i].x);
        }
        const float zero = nm == -INFINITY ? 0.0f : nm, before = __builtin_amdgcn_exp2f(m - zero);
        m = nm;
        l *= before;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] *= before;
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) {
            const float f = __builtin_amdgcn_exp2f(st[i].x - zero);
            l += f * st[i].y;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] += f * y[i][j];
        }
    }
    if constexpr (!FEW) {
        sums[tid] = x;
        if (c == 0 && grp < GROUPS) totals[grp] = make_float2(m, l);
        __syncthreads();
        if (tid >= QUADS) return;
        float top = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < GROUPS; i++) top = fmaxf(top, totals[i].x);
        m = top;
        const float zero = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
        x = (lh_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t i = 0; i < GROUPS; i++) {
            const float f = __builtin_amdgcn_exp2f(totals[i].x - zero);
            const lh_f32x4 y = sums[i * QUADS + tid];
            l += f * totals[i].y;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] += f * y[j];
        }
    }
    const float ref = fmaxf(m, sink), zero = ref == -INFINITY ? 0.0f : ref, f = __builtin_amdgcn_exp2f(m - zero);
    const float inv = l == 0.0f ? 0.0f : f / (l * f + __builtin_amdgcn_exp2f(sink - zero));
    B* out = static_cast<B*>(a.out) + (uint64_t)(tile.first + rw) * a.out_ld + (uint64_t)hd * a.dim;
#pragma unroll
    for (int j = 0; j < 4; j++) if (c + j < a.dim) out[c + j] = element_bits<DT>(x[j] * inv);
}

constexpr uint64_t kMaxWorkgroups = 0xFFFFFF;      // of 256 threads: a launch has fewer than 2^32 threads

// How a launch is cut, at most: tiles of all sequences, their parts, those that leave a record, tiles that have such.
struct Cut { uint64_t tiles, parts, records, joins; uint32_t most, least, fill, share, coarse, fixed; };
Cut cut(uint32_t tile_rows, uint32_t step, uint32_t dim, uint32_t rows, uint32_t sequences, uint32_t max_rows, uint32_t max_length, uint32_t heads, uint32_t kv_heads, uint32_t window) {
    const uint32_t R = heads / kv_heads;
    Cut c{};
    c.tiles = std::min<uint64_t>((uint64_t)rows * R / tile_rows + sequences, (uint64_t)sequences * (((uint64_t)max_rows * R + tile_rows - 1) / tile_rows));
    uint64_t steps = ((uint64_t)max_length + step - 1) / step;
    if (window) steps = std::min<uint64_t>(steps, ((uint64_t)window + tile_rows + 2 * step - 2) / step);
    c.most = (uint32_t)steps;
    c.least = (tile_rows == 16 ? 512 : 256) / step;
    // Few rows: 2048 workgroups of the 768 to 1280 that run at a time (64 tokens at 4096 to 16384 424 us, at 4000 171; with 2560 416 and 176, with 4096 418 and 180);
    // parts of 512 positions at least (a token over 32768: 27.5 us; 384 29.3, 768 30.7).  Many rows: what the chip holds at a time (256 columns: a workgroup a CU,
    // 2000 rows 71 -> 63; else two), parts of 256 (3 times 256 rows of 256 columns
    // and 29 tokens under a window of 512 27.5 us; 320 30.4).  Where the tiles alone fill
    // the chip and none is longer than 128 steps, none is cut: there is no second launch (four prompts of up to 4096 rows 225 -> 219 us, 256 tokens at 1000 178 -> 167).
    // That goes by the call's bounds.  A step recorded for 256 tokens at up to 4096 that brings one, at 4096, takes 42.5 us, where one recorded for up to 4097 takes 21.8;
    // with all 256 there, over the same pages, 307 and 315.
    c.fill = tile_rows == 16 ? 2048 : dim > 192 ? 256 : 512;
    c.share = std::max(c.fill / kv_heads, 1u);
    const uint64_t units = c.tiles * kv_heads;
    if (units >= c.fill && steps <= 128) c.least = std::max(c.least, c.most);
    while (((c.tiles * steps) >> c.coarse) + sequences > 0x7FFFFFFFull) c.coarse++;
    // nothing to measure where not even parts at least as long would fill the chip
    c.fixed = c.most <= c.least || (units < c.fill && steps / (c.fill / units) + 2 <= c.least);
    const uint64_t each = std::max<uint64_t>((steps + c.least - 1) / c.least, 1);
    c.parts = c.tiles + std::min<uint64_t>(c.tiles * (each - 1), c.share);
    if (each > 1) {
        c.records = std::min<uint64_t>(c.tiles * each, 2ull * c.share);
        c.joins = std::min<uint64_t>(c.tiles, c.share);
    }
    return c;
}
// More rows of a sequence and kv head than a tile of 16 has.  64 sequences of 2000 to 8000 positions, 8 kv heads of 128: with 4 rows of 8 heads each 256 us in tiles
// of 128 and 431 in two tiles of 16, with one row of 4 heads 493 and 438 (at 4096 to 16384).
bool takes_tiles(int dtype, uint32_t max_rows, uint32_t heads, uint32_t kv_heads) { return dtype != LH_F32 && (uint64_t)max_rows * (heads / kv_heads) > 16; }
uint32_t rows_kept(uint32_t tile_rows, uint32_t max_rows, uint32_t heads, uint32_t kv_heads) {
    return tile_rows == 16 ? (uint32_t)std::min<uint64_t>(16, (uint64_t)max_rows * (heads / kv_heads)) : tile_rows;
}
size_t cut_bytes(const Cut& c, uint32_t kept, uint32_t kv_heads, uint32_t dim) { return (size_t)c.records * kv_heads * kept * (lh_paged_padded_dim(dim) + 4) * 4; }

template <int DT, int D>
int launch_rows(lh_context* ctx, const PagedArgs& a, const Cut& c, bool tiles, const char* op, uint32_t& launches) {
    int r;
    const uint32_t wide = (uint32_t)c.parts * a.kv_heads, joins = (uint32_t)c.joins * a.kv_heads;
    launches = joins ? 2 : 1;
    if constexpr (DT != kF32) if (tiles) {
        constexpr uint32_t KT = tile_step(D);
        const size_t lds = (size_t)4 * KT * D * 2;
        if ((r = lh_raise_dynamic_lds(ctx, (const void*)paged_tiles_kernel<DT, D>, lds, op)) != LH_OK) return r;
        hipLaunchKernelGGL((paged_tiles_kernel<DT, D>), dim3(wide), dim3(256), lds, ctx->stream, a);
        if ((r = lh_check_launch(op)) != LH_OK || !joins) return r;
        // (17 rows of 8 heads over 4 at position 6000, 23 parts: the whole call 16.9 us without the turns, 13.9 with them)
        if (c.tiles * a.kv_heads * 4 < a.fill) hipLaunchKernelGGL((paged_merge_tiles_kernel<DT, D, true>), dim3(joins * (D / 4)), dim3(256), 0, ctx->stream, a);
        else hipLaunchKernelGGL((paged_merge_tiles_kernel<DT, D, false>), dim3(joins * (D / 16)), dim3(256), 0, ctx->stream, a);
        return lh_check_launch(op);
    }
    const size_t lds = (size_t)4 * 16 * (D + 4) * 4;
    if ((r = lh_raise_dynamic_lds(ctx, (const void*)paged_rows_kernel<DT, D>, lds, op)) != LH_OK) return r;
    hipLaunchKernelGGL((paged_rows_kernel<DT, D>), dim3(wide), dim3(256), lds, ctx->stream, a);
    if ((r = lh_check_launch(op)) != LH_OK || !joins) return r;
    constexpr uint32_t per = 256 / (D / 4);
    // (up to eight parts of most tiles are on their way at once; more take turns)
    if (c.tiles * a.kv_heads * 8 >= a.fill) hipLaunchKernelGGL((paged_merge_kernel<DT, D, true>), dim3(joins, (a.rows_kept + per - 1) / per), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((paged_merge_kernel<DT, D, false>), dim3(joins, a.rows_kept), dim3(256), 0, ctx->stream, a);
    return lh_check_launch(op);
}
template <int DT>
int launch_rows(lh_context* ctx, const PagedArgs& a, const Cut& c, bool tiles, const char* op, uint32_t& launches) {
    switch (lh_paged_padded_dim(a.dim)) {
        case 32: return launch_rows<DT, 32>(ctx, a, c, tiles, op, launches);
        case 64: return launch_rows<DT, 64>(ctx, a, c, tiles, op, launches);
        case 128: return launch_rows<DT, 128>(ctx, a, c, tiles, op, launches);
        case 192: return launch_rows<DT, 192>(ctx, a, c, tiles, op, launches);
        default: return launch_rows<DT, 256>(ctx, a, c, tiles, op, launches);
    }
}
}  // namespace

extern "C" {

size_t lh_paged_attention_workspace_bytes(uint32_t rows, uint32_t sequences, uint32_t max_rows, uint32_t max_length, uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    if (kv_heads == 0 || heads == 0 || heads % kv_heads || dim == 0 || dim > 256 || rows == 0 || sequences == 0 || max_rows == 0) return 0;
    size_t most = 0;                                          // of all types
    for (int dtype : {LH_BF16, LH_F32}) {
        const bool tiles = takes_tiles(dtype, max_rows, heads, kv_heads);
        const uint32_t n = tiles ? 128 : 16, kept = rows_kept(n, max_rows, heads, kv_heads);
        most = std::max(most, cut_bytes(cut(n, tiles ? tile_step(lh_paged_padded_dim(dim)) : 32, dim, rows, sequences, max_rows, max_length, heads, kv_heads, 0), kept, kv_heads, dim));
    }
    return most;
}

int lh_paged_attention_into(lh_batch* batch, const lh_buffer* q, const lh_buffer* keys, const lh_buffer* values, lh_buffer* output, int dtype, const lh_buffer* table,
                            const lh_buffer* starts, const lh_buffer* lengths, uint32_t rows, uint32_t sequences, uint32_t max_rows, uint32_t max_length, uint32_t heads,
                            uint32_t kv_heads, uint32_t dim, uint32_t pages, uint32_t page, uint32_t table_ld, uint32_t q_ld, uint32_t output_ld, float scale, uint32_t window,
                            const lh_buffer* sink, lh_buffer* workspace) {
    const char* op = "paged_attention";
    LH_REQUIRE(batch, "%s: batch is null", op);
    int r = paged_check(op, keys, values, table, starts, lengths, dtype, sequences, kv_heads, dim, pages, page, table_ld);
    if (r != LH_OK) return r;
    LH_REQUIRE(heads > 0 && heads <= 65536 && heads % kv_heads == 0, "%s: heads %u is not a multiple of kv_heads %u", op, heads, kv_heads);
    LH_REQUIRE(std::isfinite(scale * kLog2e), "%s: scale %g", op, (double)scale);      // (as the kernels have it)
    if (rows == 0) return LH_OK;
    LH_REQUIRE(max_rows > 0 && max_rows <= rows, "%s: %u rows, at most %u of a sequence", op, rows, max_rows);
    LH_REQUIRE((uint64_t)rows * heads < 0x7FFFFFFFull, "%s: %u rows of %u heads", op, rows, heads);
    const size_t size = lh_dtype_size((lh_dtype)dtype);
    const uint64_t width = (uint64_t)heads * dim;
    if ((r = paged_need_rows(op, q, "q", rows, width, q_ld, size)) != LH_OK) return r;
    if ((r = paged_need_rows(op, output, "output", rows, width, output_ld, size)) != LH_OK) return r;
    LH_REQUIRE(!paged_rows_meet(q, width, q_ld, output, width, output_ld, rows, size), "%s: q and output overlap", op);
    const size_t pool = (size_t)pages * kv_heads * page * lh_paged_padded_dim(dim) * size, out_bytes = ((size_t)(rows - 1) * output_ld + width) * size;
    for (const lh_buffer* p : {keys, values})
        LH_REQUIRE(paged_apart(p, pool, output, out_bytes), "%s: output lies inside the pages", op);
    PagedArgs a{};
    if (sink) {
        LH_NEED(sink, (size_t)heads * 4, op, "sink");
        LH_REQUIRE(((uintptr_t)sink->ptr & 3) == 0, "%s: sink has to begin at 4 bytes", op);
        a.sink = (const float*)sink->ptr;
    }
    const PagedRead read[] = {{table, (size_t)sequences * table_ld * 4, "table"}, {starts, ((size_t)sequences + 1) * 4, "starts"}, {lengths, (size_t)sequences * 4, "lengths"},
                              {sink, (size_t)heads * 4, "sink"}};
    if ((r = paged_need_apart(op, read, output, "output", width * size, (size_t)output_ld * size, rows)) != LH_OK) return r;
    const bool tiles = takes_tiles(dtype, max_rows, heads, kv_heads);
    const uint32_t tile_rows = tiles ? 128 : 16;
    const Cut c = cut(tile_rows, tiles ? tile_step(lh_paged_padded_dim(dim)) : 32, dim, rows, sequences, max_rows, max_length, heads, kv_heads, window);
    a.rows_kept = rows_kept(tile_rows, max_rows, heads, kv_heads);
    if (c.records) {
        const size_t bytes = cut_bytes(c, a.rows_kept, kv_heads, dim);
        LH_NEED(workspace, bytes, op, "workspace");
        LH_REQUIRE(paged_apart(workspace, bytes, output, out_bytes) && paged_apart(workspace, bytes, keys, pool) && paged_apart(workspace, bytes, values, pool) &&
                       paged_apart(workspace, bytes, q, ((size_t)(rows - 1) * q_ld + width) * size), "%s: workspace overlaps what the call reads or writes", op);
        if ((r = paged_need_apart(op, read, workspace, "workspace", bytes, bytes, 1)) != LH_OK) return r;
        LH_REQUIRE(((uintptr_t)workspace->ptr & 15) == 0, "%s: workspace has to begin at 16 bytes", op);
        a.partial = (float*)workspace->ptr;
    }
    LH_REQUIRE(std::max(c.parts, c.joins * 64) * kv_heads <= kMaxWorkgroups, "%s: %u rows of %u heads", op, rows, heads);
    a.q = q->ptr; a.keys = keys->ptr; a.values = values->ptr; a.out = output->ptr;
    a.plan = PagedPlan{(const uint32_t*)table->ptr, (const uint32_t*)starts->ptr, (const uint32_t*)lengths->ptr, rows, sequences, table_ld, pages, (uint32_t)__builtin_ctz(page)};
    a.q_ld = q_ld; a.out_ld = output_ld;
    a.max_rows = max_rows; a.heads = heads; a.kv_heads = kv_heads; a.dim = dim; a.window = window;
    a.capacity = (uint32_t)std::min<uint64_t>((uint64_t)table_ld * page, max_length);
    a.most = c.most; a.least = c.least; a.fill = c.fill; a.share = c.share; a.coarse = c.coarse; a.fixed = c.fixed; a.parts = (uint32_t)c.parts; a.records = (uint32_t)c.records;
    a.q_wide = (((uintptr_t)a.q | (uint64_t)q_ld * size | (uint64_t)dim * size) & 15) == 0;
    a.out_wide = (((uintptr_t)a.out | (uint64_t)output_ld * size | (uint64_t)dim * size) & 15) == 0;
    a.scale2 = scale == 0.0f ? 1.0f : std::fabs(scale) * kLog2e;
    a.negative = scale < 0.0f; a.nothing = scale == 0.0f;
    a.stream = (uint64_t)sequences * max_length * kv_heads * 2 * lh_paged_padded_dim(dim) * size > (32ull << 20);
    a.q_plain = a.q_wide && scale > 0.0f && dim == lh_paged_padded_dim(dim);
    a.group = Divisor(heads / kv_heads); a.by_heads = Divisor(kv_heads);
    uint32_t launches = 0;
    if (dtype == LH_F32) r = launch_rows<kF32>(batch->ctx, a, c, tiles, op, launches);
    else if (dtype == LH_F16) r = launch_rows<kF16>(batch->ctx, a, c, tiles, op, launches);
    else r = launch_rows<kBf16>(batch->ctx, a, c, tiles, op, launches);
    if (r == LH_OK) batch->dispatch_count += launches;
    return r;
}

}  // extern "C"
