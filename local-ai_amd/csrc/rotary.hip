// Rotary positions: pairs of a head's values turned by the position of their row, as an operation of its own and on the way of new
// keys into a paged cache.
//
// The pair (a, b) with frequency f at position p becomes amplitude * (a cos(p f) - b sin(p f), b cos(p f) + a sin(p f)).  p f is formed
// and reduced to a fraction of a turn in 64 bits (a position of 2^20 leaves 32 bits with four of the angle's), its cosine and sine are
// those of 32 bits; all of a row's heads use them, so a workgroup leaves them in LDS once per row.
//
// Memory binds it: 16384 rows of 32 heads of 128 in bf16 (268 MB) 42 us, 6.4 TB/s, 51.6 where other launches have emptied the caches; with 2 x 8 heads that go to
// pages (403 MB) 62 and 79.6.  (Stores with the streaming hint: 79.6 -> 71.5, but the attention that reads the rows next loses 21.)  A few rows: a launch's own time,
// 1.9 us, and 4.3 with the way from a row to its page (starts, table), which is three loads one behind the other.
#include "paged.hpp"
#include <algorithm>
#include <cmath>

namespace {

struct TurnArgs {
    const void* in;            // rows of `heads` heads of `dim` values: turned into `out`
    void* out;
    uint64_t in_ld, out_ld;
    uint32_t heads, dim, rot, first, rows;
    const float* frequencies;  // [rot / 2]; null: an append that turns nothing (rot is 0)
    float amplitude;
    const uint32_t* positions; // of the rows; an append has its own
    // an append
    const void *k, *v;
    void *keys, *values;
    uint64_t k_ld, v_ld;
    uint32_t kv_heads, padded;
    PagedPlan plan;
    // items of a row: of a turned head, of a key head and of a value head; of all
    uint32_t turned, key, value, items;
};

constexpr uint32_t kTurnRows = 2;          // rows of a workgroup at most (four: 16384 rows of 32 heads of 128 45.2 us, two 42.7)
constexpr uint32_t kTurnPairs = 1024;      // pairs whose cosines and sines fit

template <typename B, int V> struct ChunkOf { typedef B type __attribute__((ext_vector_type(V))); };
template <typename B> struct ChunkOf<B, 1> { typedef B type; };
template <int V, typename C> __device__ __forceinline__ auto get(const C& c, int i) { if constexpr (V == 1) return c; else return c[i]; }
template <int V, typename C, typename B> __device__ __forceinline__ void set(C& c, int i, B b) { if constexpr (V == 1) c = b; else c[i] = b; }

// An item is V neighbouring values (halves: those and their partners), V * size up to 16 bytes; V = 1 takes any size and alignment
// (neighbouring pairs: the item is a pair).  STREAM: the rows are read with the hint that nothing reads them again.
template <int DT, int V, bool HALVES, bool APPEND, bool STREAM>
__global__ __launch_bounds__(256) void turn_kernel(const TurnArgs a, uint32_t per) {
    typedef element_t<DT> B;
    typedef typename ChunkOf<B, V>::type C;
    const auto load = [](const B* p) __attribute__((always_inline)) -> C {
        if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const C*>(p));
        else return *reinterpret_cast<const C*>(p);
    };
    extern __shared__ float2 turns[];                         // [per][rot / 2]
    __shared__ uint32_t at[kTurnRows], page[kTurnRows], slot[kTurnRows];
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    const uint32_t tid = threadIdx.x, row0 = blockIdx.x * per, count = min(per, a.rows - row0), half = a.rot / 2;
    if constexpr (APPEND) {
        const uint32_t wave = tid >> 6, lane = tid & 63;
        if (wave < count) {
            const uint32_t row = row0 + wave;
            const int s = paged_sequence_of(a.plan, row, lane);
            uint32_t p = kNone, pg = kNone;
            if (s >= 0) {
                const uint32_t end = a.plan.starts[s + 1], length = a.plan.lengths[s];
                if (row < end && end <= a.plan.rows && end - row <= length) {
                    p = length - (end - row);
                    const uint32_t b = p >> a.plan.shift;
                    if (b < a.plan.table_ld) pg = a.plan.table[(size_t)s * a.plan.table_ld + b];
                    if (pg >= a.plan.pages) pg = kNone;
                }
            }
            if (lane == 0) { at[wave] = p; page[wave] = pg; slot[wave] = p & ((1u << a.plan.shift) - 1); }
        }
        __syncthreads();
    }
    for (uint32_t i = tid; i < count * half; i += 256) {
        const uint32_t r = i / half, j = i - r * half;
        const uint32_t p = APPEND ? at[r] : a.positions[row0 + r];
        const double turn = (double)p * (double)a.frequencies[j] * 0.15915494309189535;
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        turns[i] = make_float2(c * a.amplitude, s * a.amplitude);
    }
    __syncthreads();
    const uint32_t pairs = HALVES ? half / V : V == 1 ? half : a.rot / V, all = count * a.items;
    for (uint32_t it = blockIdx.y * 256 + tid; it < all; it += gridDim.y * 256) {
        const uint32_t r = it >= a.items, row = row0 + r;
        uint32_t k = it - r * a.items;
        const B* from;
        B* to;
        bool turns_it = true;
        if (!APPEND || k < a.heads * a.turned) {
            const uint32_t h = k / a.turned;
            k -= h * a.turned;
            from = static_cast<const B*>(a.in) + row * a.in_ld + (size_t)h * a.dim;
            to = static_cast<B*>(a.out) + row * a.out_ld + (size_t)h * a.dim;
            if (APPEND && at[r] == kNone) continue;
        } else {
            k -= a.heads * a.turned;
            const bool keys = k < a.kv_heads * a.key;
            if (!keys) k -= a.kv_heads * a.key;
            const uint32_t n = keys ? a.key : a.value, h = k / n;
            k -= h * n;
            if (page[r] == kNone) continue;
            from = static_cast<const B*>(keys ? a.k : a.v) + row * (keys ? a.k_ld : a.v_ld) + (size_t)h * a.dim;
            to = static_cast<B*>(keys ? a.keys : a.values) + (((((size_t)page[r] * a.kv_heads + h) << a.plan.shift) + slot[r]) * a.padded);
            turns_it = keys;
        }
        if (turns_it && k < pairs) {
            const float2* t = turns + r * half;
            if constexpr (HALVES) {
                const uint32_t d = a.first + k * V;
                C x = load(from + d), y = load(from + d + half);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float2 cs = t[k * V + i];
                    const float u = element_value<DT>(get<V>(x, i)), w = element_value<DT>(get<V>(y, i));
                    set<V>(x, i, element_bits<DT>(__builtin_fmaf(u, cs.x, -(w * cs.y))));
                    set<V>(y, i, element_bits<DT>(__builtin_fmaf(w, cs.x, u * cs.y)));
                }
                *reinterpret_cast<C*>(to + d) = x;
                *reinterpret_cast<C*>(to + d + half) = y;
            } else if constexpr (V == 1) {
                const uint32_t d = a.first + 2 * k;
                const float2 cs = t[k];
                const float u = element_value<DT>(from[d]), w = element_value<DT>(from[d + 1]);
                to[d] = element_bits<DT>(__builtin_fmaf(u, cs.x, -(w * cs.y)));
                to[d + 1] = element_bits<DT>(__builtin_fmaf(w, cs.x, u * cs.y));
            } else {
                const uint32_t d = a.first + k * V;
                C x = load(from + d);
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 cs = t[(k * V + i) / 2];
                    const float u = element_value<DT>(get<V>(x, i)), w = element_value<DT>(get<V>(x, i + 1));
                    set<V>(x, i, element_bits<DT>(__builtin_fmaf(u, cs.x, -(w * cs.y))));
                    set<V>(x, i + 1, element_bits<DT>(__builtin_fmaf(w, cs.x, u * cs.y)));
                }
                *reinterpret_cast<C*>(to + d) = x;
            }
            continue;
        }
        if (turns_it) {                                       // the columns beside the turned ones
            k -= pairs;
            const uint32_t d = k * V, c = d < a.first ? d : d + a.rot;
            C x = 0;
            if (c < a.dim) x = load(from + c);
            *reinterpret_cast<C*>(to + c) = x;
        } else {
            const uint32_t c = k * V;
            C x = 0;
            if (c < a.dim) x = load(from + c);
            *reinterpret_cast<C*>(to + c) = x;
        }
    }
}

template <int DT, int V, bool APPEND, bool STREAM = false>
int launch_turn(lh_context* ctx, TurnArgs& a, uint32_t pairing, const char* op) {
    const bool halves = pairing == LH_ROTARY_HALVES;
    const uint32_t pairs = halves ? a.rot / 2 / V : V == 1 ? a.rot / 2 : a.rot / V;
    a.turned = pairs + (a.dim - a.rot) / V;
    a.key = a.turned + (a.padded - a.dim) / V;
    a.value = a.padded / V;
    const uint64_t items = (uint64_t)a.heads * a.turned + (APPEND ? (uint64_t)a.kv_heads * (a.key + a.value) : 0);
    LH_REQUIRE(items * kTurnRows < 0x7FFFFFFFull, "%s: rows of %u heads", op, a.heads);
    a.items = (uint32_t)items;
    uint32_t per = kTurnRows;
    while (per > 1 && ((a.rows + per - 1) / per < 2048 || per * (a.rot / 2) > kTurnPairs)) per /= 2;
    const uint32_t groups = (a.rows + per - 1) / per, split = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(1, items * per / 2048), 64);
    LH_REQUIRE((uint64_t)groups * split <= 0xFFFFFF, "%s: %u rows", op, a.rows);      // a launch has fewer than 2^32 threads
    const size_t lds = (size_t)per * (a.rot / 2) * sizeof(float2);
    if (halves) hipLaunchKernelGGL((turn_kernel<DT, V, true, APPEND, STREAM>), dim3(groups, split), dim3(256), lds, ctx->stream, a, per);
    else hipLaunchKernelGGL((turn_kernel<DT, V, false, APPEND, STREAM>), dim3(groups, split), dim3(256), lds, ctx->stream, a, per);
    return lh_check_launch(op);
}

template <int DT, int V, bool APPEND>
int launch_wide(lh_context* ctx, TurnArgs& a, uint32_t pairing, bool stream, const char* op) {
    return stream ? launch_turn<DT, V, APPEND, true>(ctx, a, pairing, op) : launch_turn<DT, V, APPEND>(ctx, a, pairing, op);
}

// The widest items that every row, head and part begins and ends with.
template <bool APPEND>
int launch_turn(lh_context* ctx, TurnArgs& a, int dtype, uint32_t pairing, const char* op) {
    const size_t size = lh_dtype_size((lh_dtype)dtype);
    uintptr_t bytes = (uintptr_t)a.in | (uintptr_t)a.out | (uintptr_t)a.k | (uintptr_t)a.v;      // (pages begin at 16)
    uint64_t values = a.first | a.dim | (pairing == LH_ROTARY_HALVES ? a.rot / 2 : a.rot) | a.k_ld | a.v_ld | (a.heads ? a.in_ld | a.out_ld : 0);
    bytes |= values * size;
    const uint32_t wide = (bytes & 15) == 0 ? 16 / size : (bytes & (2 * size - 1)) == 0 ? 2 : 1;
    // More than stays near the chip: 16384 rows of 32 + 2 x 8 heads of 128 80 -> 64 us, their query heads 45 -> 43; 4500 rows of 16 + 2 x 4 heads, which a
    // program's last launch has left there, 14.5 -> 19.
    const bool stream = (uint64_t)a.rows * (a.heads + 2ull * a.kv_heads) * a.dim * size * 2 > (256ull << 20);
    if (dtype == LH_F32) return wide == 4 ? launch_wide<kF32, 4, APPEND>(ctx, a, pairing, stream, op) : wide == 2 ? launch_turn<kF32, 2, APPEND>(ctx, a, pairing, op)
                                                                                                                 : launch_turn<kF32, 1, APPEND>(ctx, a, pairing, op);
    if (dtype == LH_F16) return wide == 8 ? launch_wide<kF16, 8, APPEND>(ctx, a, pairing, stream, op) : wide == 2 ? launch_turn<kF16, 2, APPEND>(ctx, a, pairing, op)
                                                                                                                 : launch_turn<kF16, 1, APPEND>(ctx, a, pairing, op);
    return wide == 8 ? launch_wide<kBf16, 8, APPEND>(ctx, a, pairing, stream, op) : wide == 2 ? launch_turn<kBf16, 2, APPEND>(ctx, a, pairing, op)
                                                                                              : launch_turn<kBf16, 1, APPEND>(ctx, a, pairing, op);
}

int check_rotation(const char* op, const lh_buffer* frequencies, uint32_t dim, uint32_t rot, uint32_t first, uint32_t pairing) {
    LH_REQUIRE(pairing == LH_ROTARY_PAIRS || pairing == LH_ROTARY_HALVES, "%s: pairing %u", op, pairing);
    LH_REQUIRE(rot % 2 == 0 && rot <= dim && first <= dim - rot, "%s: columns %u .. %llu turned of %u", op, first, (unsigned long long)first + rot, dim);
    LH_NEED(frequencies, (size_t)rot / 2 * 4, op, "frequencies");
    LH_REQUIRE(((uintptr_t)frequencies->ptr & 3) == 0, "%s: frequencies have to begin at 4 bytes", op);
    return LH_OK;
}

}  // namespace

extern "C" {

int lh_rotary_frequencies(uint32_t rot, float base, uint32_t scaling, float factor, float original, float fast, float slow, float* frequencies, float* amplitude) {
    const char* op = "rotary_frequencies";
    LH_REQUIRE(frequencies && amplitude, "%s: null argument", op);
    LH_REQUIRE(rot >= 2 && rot % 2 == 0 && rot <= 4096, "%s: %u turned columns", op, rot);
    LH_REQUIRE(base > 1.0f && std::isfinite(base), "%s: base %g", op, (double)base);
    LH_REQUIRE(scaling == LH_ROTARY_PLAIN || scaling == LH_ROTARY_LINEAR || scaling == LH_ROTARY_BY_PARTS, "%s: scaling %u", op, scaling);
    LH_REQUIRE(scaling == LH_ROTARY_PLAIN || (factor >= 1.0f && std::isfinite(factor)), "%s: factor %g", op, (double)factor);
    const bool parts = scaling == LH_ROTARY_BY_PARTS;
    LH_REQUIRE(!parts || (original >= 1.0f && std::isfinite(original) && slow > 0.0f && fast > slow && std::isfinite(fast)), "%s: parts between %g and %g turns in %g positions", op,
               (double)slow, (double)fast, (double)original);
    const double two_pi = 6.283185307179586476925, n = rot;
    // the index whose frequency makes `turns` turns in the original length
    const auto index = [&](double turns) { return n * std::log((double)original / (turns * two_pi)) / (2.0 * std::log((double)base)); };
    double lo = 0.0, hi = 1.0;
    if (parts) {
        lo = std::max(std::floor(index(fast)), 0.0);
        hi = std::min(std::ceil(index(slow)), n - 1.0);
        if (hi <= lo) hi = lo + 0.001;
    }
    for (uint32_t i = 0; i < rot / 2; i++) {
        const double f = std::pow((double)base, -2.0 * i / n);
        double keep = scaling == LH_ROTARY_PLAIN ? 1.0 : 0.0;      // the share that is not stretched
        if (parts) keep = 1.0 - std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
        frequencies[i] = (float)(f * keep + (scaling == LH_ROTARY_PLAIN ? 0.0 : f / factor * (1.0 - keep)));
    }
    *amplitude = parts ? (float)(0.1 * std::log((double)factor) + 1.0) : 1.0f;
    return LH_OK;
}

int lh_rotary_rows_into(lh_batch* batch, const lh_buffer* input, lh_buffer* output, int dtype, const lh_buffer* positions, const lh_buffer* frequencies, float amplitude,
                        uint32_t rows, uint32_t heads, uint32_t dim, uint32_t rot, uint32_t first, uint32_t pairing, uint32_t input_ld, uint32_t output_ld) {
    const char* op = "rotary_rows";
    LH_REQUIRE(batch, "%s: batch is null", op);
    LH_REQUIRE(dtype == LH_F16 || dtype == LH_BF16 || dtype == LH_F32, "%s: dtype %d", op, dtype);
    LH_REQUIRE(dim > 0 && dim <= 1024 && heads <= 65536, "%s: %u heads of %u", op, heads, dim);
    int r = check_rotation(op, frequencies, dim, rot, first, pairing);
    if (r != LH_OK) return r;
    if (rows == 0 || heads == 0) return LH_OK;
    const size_t size = lh_dtype_size((lh_dtype)dtype);
    const uint64_t width = (uint64_t)heads * dim;
    if ((r = paged_need_rows(op, input, "input", rows, width, input_ld, size)) != LH_OK) return r;
    if ((r = paged_need_rows(op, output, "output", rows, width, output_ld, size)) != LH_OK) return r;
    LH_NEED(positions, (size_t)rows * 4, op, "positions");
    LH_REQUIRE(((uintptr_t)positions->ptr & 3) == 0, "%s: positions have to begin at 4 bytes", op);
    LH_REQUIRE((input->ptr == output->ptr && input_ld == output_ld) || !paged_rows_meet(input, width, input_ld, output, width, output_ld, rows, size),
               "%s: input and output overlap and are not the same", op);
    const PagedRead read[] = {{positions, (size_t)rows * 4, "positions"}, {frequencies, (size_t)rot / 2 * 4, "frequencies"}};
    if ((r = paged_need_apart(op, read, output, "output", width * size, (size_t)output_ld * size, rows)) != LH_OK) return r;
    TurnArgs a{};
    a.in = input->ptr; a.out = output->ptr; a.in_ld = input_ld; a.out_ld = output_ld;
    a.heads = heads; a.dim = dim; a.rot = rot; a.first = first; a.rows = rows; a.padded = dim;
    a.frequencies = (const float*)frequencies->ptr; a.amplitude = amplitude; a.positions = (const uint32_t*)positions->ptr;
    r = launch_turn<false>(batch->ctx, a, dtype, pairing, op);
    if (r == LH_OK) batch->dispatch_count++;
    return r;
}

uint32_t lh_paged_padded_dim(uint32_t dim) { return dim <= 32 ? 32u : dim <= 64 ? 64u : dim <= 128 ? 128u : dim <= 192 ? 192u : 256u; }

int lh_paged_append_into(lh_batch* batch, const lh_buffer* k, const lh_buffer* v, int dtype, lh_buffer* keys, lh_buffer* values, const lh_buffer* table, const lh_buffer* starts,
                         const lh_buffer* lengths, uint32_t rows, uint32_t sequences, uint32_t kv_heads, uint32_t dim, uint32_t pages, uint32_t page, uint32_t table_ld,
                         uint32_t k_ld, uint32_t v_ld, const lh_buffer* frequencies, float amplitude, uint32_t rot, uint32_t first, uint32_t pairing, const lh_buffer* q,
                         lh_buffer* q_output, uint32_t heads, uint32_t q_ld, uint32_t q_output_ld) {
    const char* op = "paged_append";
    LH_REQUIRE(batch, "%s: batch is null", op);
    int r = paged_check(op, keys, values, table, starts, lengths, dtype, sequences, kv_heads, dim, pages, page, table_ld);
    if (r != LH_OK) return r;
    LH_REQUIRE(frequencies || rot == 0, "%s: %u turned columns without frequencies", op, rot);
    if (frequencies && (r = check_rotation(op, frequencies, dim, rot, first, pairing)) != LH_OK) return r;
    LH_REQUIRE((q == nullptr) == (q_output == nullptr) && (q != nullptr) == (heads > 0), "%s: queries, their output and their heads come together", op);
    LH_REQUIRE(heads <= 65536, "%s: %u heads", op, heads);
    if (rows == 0) return LH_OK;
    const size_t size = lh_dtype_size((lh_dtype)dtype);
    const uint64_t kvw = (uint64_t)kv_heads * dim, qw = (uint64_t)heads * dim;
    if ((r = paged_need_rows(op, k, "k", rows, kvw, k_ld, size)) != LH_OK) return r;
    if ((r = paged_need_rows(op, v, "v", rows, kvw, v_ld, size)) != LH_OK) return r;
    if (q) {
        if ((r = paged_need_rows(op, q, "q", rows, qw, q_ld, size)) != LH_OK) return r;
        if ((r = paged_need_rows(op, q_output, "q_output", rows, qw, q_output_ld, size)) != LH_OK) return r;
        LH_REQUIRE((q->ptr == q_output->ptr && q_ld == q_output_ld) || !paged_rows_meet(q, qw, q_ld, q_output, qw, q_output_ld, rows, size),
                   "%s: q and q_output overlap and are not the same", op);
        LH_REQUIRE(!paged_rows_meet(k, kvw, k_ld, q_output, qw, q_output_ld, rows, size) && !paged_rows_meet(v, kvw, v_ld, q_output, qw, q_output_ld, rows, size),
                   "%s: q_output lies over k or v", op);
    }
    const size_t pool = (size_t)pages * kv_heads * page * lh_paged_padded_dim(dim) * size;
    const auto apart = [&](const lh_buffer* b, uint64_t width, uint32_t ld, const lh_buffer* p) { return paged_apart(b, ((size_t)(rows - 1) * ld + width) * size, p, pool); };
    for (const lh_buffer* p : {(const lh_buffer*)keys, (const lh_buffer*)values})
        LH_REQUIRE(apart(k, kvw, k_ld, p) && apart(v, kvw, v_ld, p) && (!q || (apart(q, qw, q_ld, p) && apart(q_output, qw, q_output_ld, p))), "%s: the rows lie inside the pages", op);
    LH_REQUIRE(paged_apart(keys, pool, values, pool), "%s: keys and values have pages of their own", op);
    const PagedRead read[] = {{table, (size_t)sequences * table_ld * 4, "table"}, {starts, ((size_t)sequences + 1) * 4, "starts"}, {lengths, (size_t)sequences * 4, "lengths"},
                              {frequencies, (size_t)rot / 2 * 4, "frequencies"}};
    if ((r = paged_need_apart(op, read, keys, "keys", pool, pool, 1)) != LH_OK) return r;
    if ((r = paged_need_apart(op, read, values, "values", pool, pool, 1)) != LH_OK) return r;
    if (q && (r = paged_need_apart(op, read, q_output, "q_output", qw * size, (size_t)q_output_ld * size, rows)) != LH_OK) return r;
    TurnArgs a{};
    if (q) { a.in = q->ptr; a.out = q_output->ptr; a.in_ld = q_ld; a.out_ld = q_output_ld; }
    a.heads = heads; a.dim = dim; a.rot = rot; a.first = rot ? first : 0; a.rows = rows;
    a.frequencies = frequencies ? (const float*)frequencies->ptr : nullptr; a.amplitude = amplitude;
    a.k = k->ptr; a.v = v->ptr; a.keys = keys->ptr; a.values = values->ptr; a.k_ld = k_ld; a.v_ld = v_ld;
    a.kv_heads = kv_heads; a.padded = lh_paged_padded_dim(dim);
    a.plan = PagedPlan{(const uint32_t*)table->ptr, (const uint32_t*)starts->ptr, (const uint32_t*)lengths->ptr, rows, sequences, table_ld, pages, (uint32_t)__builtin_ctz(page)};
    r = launch_turn<true>(batch->ctx, a, dtype, rot ? pairing : (uint32_t)LH_ROTARY_PAIRS, op);
    if (r == LH_OK) batch->dispatch_count++;
    return r;
}

}  // extern "C"
