// What the kernels over paged caches share (rotary.hip: rows that go to pages; paged_attention.hip: queries over them): the element
// types, and where the rows of a step belong.
#pragma once
#include "float_ops.hpp"

namespace {

constexpr int kF16 = LH_F16, kF32 = LH_F32, kBf16 = LH_BF16;

// Elements as raw bits; copies move the bits.
template <int DT> struct PagedElement { typedef uint16_t type; };
template <> struct PagedElement<kF32> { typedef uint32_t type; };
template <int DT> using element_t = typename PagedElement<DT>::type;

template <int DT>
__device__ __forceinline__ float element_value(element_t<DT> b) {
    if constexpr (DT == kF32) return __builtin_bit_cast(float, b);
    else if constexpr (DT == kF16) return lh_h2f(b);
    else return lh_bf2f(b);
}
template <int DT>
__device__ __forceinline__ element_t<DT> element_bits(float v) {      // round to nearest even
    if constexpr (DT == kF32) return __builtin_bit_cast(uint32_t, v);
    else if constexpr (DT == kF16) return lh_f2h(v);
    else return lh_f2bf(v);
}

// The sequences of a step and their pages, all in device memory.  Nothing that stands there can lead a kernel out of its buffers.
struct PagedPlan {
    const uint32_t* table;     // [sequences][table_ld]
    const uint32_t* starts;    // [sequences + 1]
    const uint32_t* lengths;   // [sequences]
    uint32_t rows, sequences, table_ld, pages, shift;   // shift: log2 of a page's positions
};

// The last sequence that starts at or before `row`, found by whole waves, 64 ways at a time; -1 without one.
__device__ __forceinline__ int paged_sequence_of(const PagedPlan& p, uint32_t row, uint32_t lane) {
    uint32_t lo = 0, n = p.sequences;
    while (true) {
        const uint32_t step = (n + 63) / 64, at = lane * step;
        const bool before = at < n && p.starts[lo + at] <= row;
        const uint64_t all = __ballot(before);
        if (all == 0) return lo == 0 ? -1 : (int)lo;
        const uint32_t last = 63 - __builtin_clzll(all);
        lo += last * step;
        n = min(step, n - last * step);
        if (step == 1) return (int)lo;
    }
}

// Host side: validates what every operation over pages gets.
inline int paged_check(const char* op, const lh_buffer* keys, const lh_buffer* values, const lh_buffer* table, const lh_buffer* starts, const lh_buffer* lengths, int dtype,
                       uint32_t sequences, uint32_t kv_heads, uint32_t dim, uint32_t pages, uint32_t page, uint32_t table_ld) {
    LH_REQUIRE(dtype == LH_F16 || dtype == LH_BF16 || dtype == LH_F32, "%s: dtype %d", op, dtype);
    LH_REQUIRE(kv_heads > 0 && kv_heads <= 1024, "%s: %u kv heads", op, kv_heads);
    LH_REQUIRE(dim > 0 && dim <= 256, "%s: heads of %u dimensions, pages take 1 to 256", op, dim);
    LH_REQUIRE(page >= 16 && page <= 1024 && (page & (page - 1)) == 0, "%s: pages of %u positions, a power of two from 16 to 1024 is wanted", op, page);
    LH_REQUIRE(pages > 0 && table_ld > 0 && (uint64_t)table_ld * page <= 0x7FFFFFFFull, "%s: %u pages, %u to a sequence", op, pages, table_ld);
    LH_REQUIRE(sequences > 0 && sequences <= (1u << 20), "%s: %u sequences", op, sequences);
    const size_t bytes = (size_t)pages * kv_heads * page * lh_paged_padded_dim(dim) * lh_dtype_size((lh_dtype)dtype);
    LH_NEED(keys, bytes, op, "keys");
    LH_NEED(values, bytes, op, "values");
    LH_NEED(table, (size_t)sequences * table_ld * 4, op, "table");
    LH_NEED(starts, ((size_t)sequences + 1) * 4, op, "starts");
    LH_NEED(lengths, (size_t)sequences * 4, op, "lengths");
    LH_REQUIRE(((((uintptr_t)keys->ptr) | ((uintptr_t)values->ptr)) & 15) == 0, "%s: pages have to begin at 16 bytes", op);
    LH_REQUIRE(((((uintptr_t)table->ptr) | ((uintptr_t)starts->ptr) | ((uintptr_t)lengths->ptr)) & 3) == 0, "%s: table, starts and lengths have to begin at 4 bytes", op);
    return LH_OK;
}

// `rows` rows of `width` values, `ld` apart, at the start of `b`.
inline int paged_need_rows(const char* op, const lh_buffer* b, const char* name, uint32_t rows, uint64_t width, uint32_t ld, size_t size) {
    LH_REQUIRE(ld >= width, "%s: rows of %s are %u values apart and have %llu", op, name, ld, (unsigned long long)width);
    LH_NEED(b, rows ? ((size_t)(rows - 1) * ld + width) * size : 0, op, name);
    LH_REQUIRE(((uintptr_t)b->ptr & (size - 1)) == 0, "%s: %s has to begin at a value", op, name);
    return LH_OK;
}
inline bool paged_apart(const lh_buffer* a, size_t abytes, const lh_buffer* b, size_t bbytes) {
    return (uintptr_t)a->ptr + abytes <= (uintptr_t)b->ptr || (uintptr_t)b->ptr + bbytes <= (uintptr_t)a->ptr;
}
// Whether two sets of such rows share memory.  Rows at one distance may lie side by side.
inline bool paged_rows_meet(const lh_buffer* a, uint64_t awidth, uint32_t ald, const lh_buffer* b, uint64_t bwidth, uint32_t bld, uint32_t rows, size_t size) {
    if (rows == 0 || awidth == 0 || bwidth == 0) return false;
    const uintptr_t a0 = (uintptr_t)a->ptr, b0 = (uintptr_t)b->ptr;
    if (a0 + ((size_t)(rows - 1) * ald + awidth) * size <= b0 || b0 + ((size_t)(rows - 1) * bld + bwidth) * size <= a0) return false;
    if (ald != bld) return true;
    const size_t ld = (size_t)ald * size, d = b0 >= a0 ? (b0 - a0) % ld : (ld - (a0 - b0) % ld) % ld;    // where b's row begins in a's
    return d < awidth * size || d + bwidth * size > ld;
}
// Whether `bytes` at the start of b share memory with rows of `width` bytes, `ld` bytes apart, from `out` on.
inline bool paged_meets(const lh_buffer* b, size_t bytes, const lh_buffer* out, size_t width, size_t ld, uint32_t rows) {
    if (bytes == 0 || rows == 0 || width == 0) return false;
    const uintptr_t b0 = (uintptr_t)b->ptr, o0 = (uintptr_t)out->ptr;
    if (b0 + bytes <= o0 || o0 + (size_t)(rows - 1) * ld + width <= b0) return false;
    if (b0 < o0) return true;
    const size_t at = (b0 - o0) % ld;                         // between two rows there is room for others' data
    return at < width || at + bytes > ld;
}
// What a step's plan is read from, beside the rows: none of it may lie where a kernel writes.
struct PagedRead { const lh_buffer* b; size_t bytes; const char* name; };
template <size_t N>
inline int paged_need_apart(const char* op, const PagedRead (&read)[N], const lh_buffer* out, const char* name, size_t width, size_t ld, uint32_t rows) {
    for (const PagedRead& r : read) LH_REQUIRE(!r.b || !paged_meets(r.b, r.bytes, out, width, ld, rows), "%s: %s lies over %s", op, name, r.name);
    return LH_OK;
}

}  // namespace
