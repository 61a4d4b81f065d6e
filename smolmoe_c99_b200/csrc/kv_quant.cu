// Writing the 8-bit key/value cache and reading it back (the format: kv_quant.cuh).
//
// Both are bound by memory: a thread takes 8 or 16 values of a row at a time (16 or 32 bytes in, 8 or 16 out, or the other way)
// and several rows at once; the lanes that share a row find its largest magnitude with shuffles, so a value is read once and
// written once.
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "kv_quant.cuh"
#include "launch.cuh"

namespace sm {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct StoreArgs {
    const void* packed[2];       // keys, values [T, kv_heads, head_dim]
    void* rows[2];               // what the cache then stands for, laid out like packed (nullable)
    uint8_t* codes[2];
    uint8_t* scales[2];
    const int32_t* positions;    // [T]
    const int32_t* token_slot;   // [T]
    QuantPages pages;
    int kv_heads, head_dim;
    unsigned rows_of_each;       // T * kv_heads
    int* error;
};

// One row per group of threads (a power of two of them), V values each; blockIdx.y: keys or values. A thread does kStoreRows
// rows, so that as many loads are under way together. What a row costs whatever its length (its token, its page, its
// place) weighs as much as 16 values do, so a thread takes 16 of bfloat16 where the head size allows (prompts of 22,000 tokens of 4
// heads of 128 written, and 61,000 positions read back: 48 us, with 8 values a thread 55), and 8 of float (prompts of up to 2,000
// tokens: 8.4 us, with 16 9.0).
constexpr int kStoreRows = 2;

// V values of a row as they were loaded: 16-byte pieces of a type.
template <typename T, int V>
struct Piece {
    static constexpr int N = V * sizeof(T) / 16;
    uint4 raw[N];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& r = raw[i / 4];
        return i % 4 == 0 ? r.x : i % 4 == 1 ? r.y : i % 4 == 2 ? r.z : r.w;
    }
    __device__ __forceinline__ float value(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(word(i));
        return i % 2 == 0 ? __uint_as_float(word(i / 2) << 16) : __uint_as_float(word(i / 2) & 0xffff0000u);
    }
    // Magnitudes as whole numbers, whose order is theirs: of float one a word, of bfloat16 two.
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b); }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N * 4; ++i) m = larger(m, word(i) & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu));
        return m;
    }
    static __device__ __forceinline__ uint32_t as_float_bits(uint32_t m) { return sizeof(T) == 4 ? m : max(m & 0xffff0000u, m << 16); }
};

template <typename T, int FMT, int V>
__global__ void __launch_bounds__(kThreads) kv_quant_store_kernel(StoreArgs a, int log_lanes, unsigned per_kv_head) {
    pdl_wait();                  // the rows come from the kernel before
    pdl_launch_dependents();
    const int lanes = 1 << log_lanes, per_block = kThreads >> log_lanes;
    const unsigned row0 = blockIdx.x * (per_block * kStoreRows) + (threadIdx.x >> log_lanes);
    const int part = threadIdx.x & (lanes - 1);
    // (chosen, not indexed: an index that is not a constant would put the arguments into local memory)
    const bool keys = blockIdx.y == 0;
    const T* packed = (const T*)(keys ? a.packed[0] : a.packed[1]);
    T* rows = (T*)(keys ? a.rows[0] : a.rows[1]);
    uint8_t* codes = keys ? a.codes[0] : a.codes[1];
    uint8_t* scales = keys ? a.scales[0] : a.scales[1];
    Piece<T, V> x[kStoreRows];
    int at_token[kStoreRows], at_slot[kStoreRows], kv_head[kStoreRows];
    bool mine[kStoreRows];
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) {
        const unsigned row = row0 + u * per_block;
        const bool live = row < a.rows_of_each;
        mine[u] = live && part * V < a.head_dim;
        x[u].clear();
        if (mine[u]) x[u].load(packed + (size_t)row * a.head_dim + part * V);
        // row / kv_heads, by the floor of 2^32 / kv_heads (2^32 - 1 for one head): at most one too few
        unsigned t = live ? __umulhi(row, per_kv_head) : 0, h = live ? row - t * (unsigned)a.kv_heads : 0;
        if (h >= (unsigned)a.kv_heads) { ++t; h -= (unsigned)a.kv_heads; }
        kv_head[u] = (int)h;
        at_token[u] = a.positions[t];
        at_slot[u] = a.token_slot[t];
    }
    int page[kStoreRows];
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) page[u] = at_token[u] < 0 ? -1 : a.pages.at(at_slot[u], at_token[u] / kPageSize);
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) {
        const unsigned row = row0 + u * per_block;
        uint32_t m = x[u].largest();
        for (int o = lanes >> 1; o > 0; o >>= 1) m = Piece<T, V>::larger(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!mine[u]) continue;
        const int byte = scale_byte<FMT>(Piece<T, V>::as_float_bits(m));
        uint32_t code[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) code[i] = 0;
        if (byte != kNoScale) {
            const float up = power_of_two(127 - byte);
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                code[i] = encode4<FMT>(x[u].value(4 * i) * up, x[u].value(4 * i + 1) * up, x[u].value(4 * i + 2) * up, x[u].value(4 * i + 3) * up);
        }
        if (page[u] >= 0) {
            const size_t cell = ((size_t)page[u] * a.kv_heads + kv_head[u]) * kPageSize + at_token[u] % kPageSize;
            uint8_t* dst = codes + cell * a.head_dim + part * V;
            if (V == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(code[0], code[1], code[V / 4 - 2], code[V / 4 - 1]);
            else *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
            if (part == 0) scales[cell] = (uint8_t)byte;
        } else if (a.error) {
            atomicExch(a.error, kBadPlaceInStore);
        }
        if (rows != nullptr) {
            const float scale = scale_of(byte);
#pragma unroll
            for (int i = 0; i < V / 8; ++i) {
                float v[4], w[4];
                decode4<FMT>(code[2 * i], v);
                decode4<FMT>(code[2 * i + 1], w);
                const float y[8] = {v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale, w[0] * scale, w[1] * scale, w[2] * scale, w[3] * scale};
                store8(rows + (size_t)row * a.head_dim + part * V + 8 * i, y);
            }
        }
    }
}

struct LoadArgs {
    const uint8_t* codes[2];
    const uint8_t* scales[2];
    void* out[2];                // [room, kv_heads, kPageSize, head_dim]
    int32_t* out_table;          // [slots, pages]: where a slot's pages lie in `out` (nullable)
    const int32_t* slot_ids;     // [sequences]
    const int32_t* seq_ends;     // [sequences]
    QuantPages table;
    int kv_heads, head_dim, seqs, pages, whole;
    long long room;              // pages of `out`
    const int32_t* cu;           // [sequences + 1] (not read where all is read back whole)
    int skip_new;                // sequences that bring at most this many tokens are left out
    int attend, window;          // see kv_quant_load in kernels.h
    int* error;
};

// The sequence that is number `rank` of those that are read back (-1: there is none), its pages, and how many pages the ones before
// it take. Each warp goes through the step's sequences by itself, 32 at once.
struct SequenceRead {
    int seq;
    long long before;
    PagesRead pages;
};
__device__ __forceinline__ SequenceRead find_sequence(const LoadArgs& a, int rank) {
    const int lane = threadIdx.x & 31;
    int seen = 0;
    long long before = 0;
    for (int i0 = 0; i0 < a.seqs; i0 += 32) {
        const int i = i0 + lane, n = i < a.seqs ? a.cu[i + 1] - a.cu[i] : -1, end = i < a.seqs ? a.seq_ends[i] : 0;
        const PagesRead p = pages_read(end - n, end, a.window, a.pages);
        const unsigned read = __ballot_sync(0xffffffffu, n > a.skip_new);
        const int mine = n > a.skip_new ? seen + __popc(read & ((1u << lane) - 1)) : -1;
        before += __reduce_add_sync(0xffffffffu, mine >= 0 && mine < rank ? p.count : 0);
        const unsigned hit = __ballot_sync(0xffffffffu, mine == rank);
        if (hit) {
            const int at = __ffs(hit) - 1;
            return {i0 + at, before, {__shfl_sync(0xffffffffu, p.first, at), __shfl_sync(0xffffffffu, p.count, at)}};
        }
        seen += __popc(read);
    }
    return {-1, 0, {0, 0}};
}

// A CTA reads one page (blockIdx.x, from the first that is read back) of one sequence (blockIdx.y, of those that are read back),
// keys or values (blockIdx.z): a page's kv heads lie one behind the other in the pools and in the output, so this is one run of
// bytes and one of values, 8 of them a thread and kLoadSteps such pieces under way together. Positions at and past the sequence's
// end read as zero. `whole`: every sequence has `pages` pages of the output, zeros past its end; otherwise they lie one behind
// the other, each as many as it holds.
constexpr int kLoadSteps = 4;

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) kv_quant_load_kernel(LoadArgs a) {
    pdl_wait();                  // the cache may have been written by the kernel before
    pdl_launch_dependents();
    const int which = blockIdx.z;
    if (a.whole && which == 1 && blockIdx.y == 0)       // slots that are not the step's are given a page that exists
        for (int slot = threadIdx.x; slot < a.table.slots; slot += kThreads) {
            bool named = false;
            for (int i = 0; i < a.seqs; ++i) named |= a.slot_ids[i] == slot;
            if (!named) a.out_table[(size_t)slot * a.pages + blockIdx.x] = 0;
        }
    const SequenceRead r = a.whole ? SequenceRead{(int)blockIdx.y, (long long)blockIdx.y * a.pages, {0, a.pages}} : find_sequence(a, blockIdx.y);
    if (r.seq < 0) return;
    const int slot = a.slot_ids[r.seq], end = a.seq_ends[r.seq], page = r.pages.first + blockIdx.x;
    // (what does not fit is left out)
    if ((unsigned)slot >= (unsigned)a.table.slots || end > a.pages * kPageSize || r.before + r.pages.count > a.room) {
        if (a.error && threadIdx.x == 0) atomicExch(a.error, kBadPlaceInLoad);
        if ((unsigned)slot >= (unsigned)a.table.slots || r.before + r.pages.count > a.room) return;
    }
    if ((int)blockIdx.x >= r.pages.count) return;
    const long long to = r.before + blockIdx.x;
    if (which == 0 && threadIdx.x == 0 && a.out_table) a.out_table[(size_t)slot * a.pages + page] = (int)to;
    const int live = min(end - page * kPageSize, kPageSize);      // positions of the page that the sequence holds
    const int held = live > 0 ? a.table.at(slot, page) : -1;
    if (live > 0 && held < 0 && a.error && threadIdx.x == 0) atomicExch(a.error, kBadPlaceInLoad);
    const int parts = a.head_dim / 8, total = a.kv_heads * kPageSize * parts;      // pieces of 8 values: of a row, of the page
    const size_t cell0 = held < 0 ? 0 : (size_t)held * a.kv_heads * kPageSize;
    const uint8_t* codes = a.codes[which] + cell0 * a.head_dim;
    T* out = (T*)a.out[which] + (size_t)to * a.kv_heads * kPageSize * a.head_dim;
    for (int base = threadIdx.x; base < total; base += kThreads * kLoadSteps) {
        uint2 raw[kLoadSteps];
        int byte[kLoadSteps];
#pragma unroll
        for (int u = 0; u < kLoadSteps; ++u) {
            const int i = base + u * kThreads, row = i / parts;
            raw[u] = make_uint2(0, 0);
            byte[u] = 0;
            if (i < total && held >= 0 && row % kPageSize < live) {
                raw[u] = *reinterpret_cast<const uint2*>(codes + (size_t)i * 8);
                byte[u] = a.scales[which][cell0 + row];
                if (a.attend) {
                    if (which == 0 && a.scales[1][cell0 + row] == kNoScale) byte[u] = kNoScale;
                    if (which == 1 && byte[u] == kNoScale) byte[u] = 0;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kLoadSteps; ++u) {
            const int i = base + u * kThreads;
            if (i >= total) break;
            const float scale = scale_of(byte[u]);
            const bool none = byte[u] == kNoScale;      // (also where the codes are another row's: a key whose value has no scale)
            float v[4], w[4], y[8];
            decode4<FMT>(raw[u].x, v);
            decode4<FMT>(raw[u].y, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = none ? __int_as_float(0x7fffffff) : v[e] * scale;
                y[4 + e] = none ? __int_as_float(0x7fffffff) : w[e] * scale;
            }
            store8(out + (size_t)i * 8, y);
        }
    }
}

void check_pools(const char* who, const QuantPools& p) {
    if (p.kv_heads <= 0 || p.head_dim <= 0 || p.head_dim % 8 || p.head_dim > 256)
        throw std::invalid_argument(std::string(who) + ": head_dim " + std::to_string(p.head_dim) + " is not a multiple of 8 up to 256");
    if (p.fmt != QUANT_FP8 && p.fmt != QUANT_INT8) throw std::invalid_argument(std::string(who) + ": unknown format " + std::to_string(p.fmt));
    if (((uintptr_t)p.k_codes | (uintptr_t)p.v_codes) & 7) throw std::invalid_argument(std::string(who) + ": pools must be 8-byte aligned");
}

}  // namespace

void kv_quant_store(const QuantPools& p, const void* k_packed, const void* v_packed, DType dt, int T, void* k_rows, void* v_rows,
                    const int32_t* positions, const int32_t* token_slot, int* error, cudaStream_t stream) {
    if (T <= 0) return;
    check_pools("kv_quant_store", p);
    if (((uintptr_t)k_packed | (uintptr_t)v_packed | (uintptr_t)k_rows | (uintptr_t)v_rows) & 15)
        throw std::invalid_argument("kv_quant_store: rows must be 16-byte aligned");
    if ((long long)T * p.kv_heads > 0x7fffffffll) throw std::invalid_argument("kv_quant_store: more than 2^31 rows in one call");
    const int each = dt == F32 || p.head_dim % 16 || ((uintptr_t)p.k_codes | (uintptr_t)p.v_codes) & 15 ? 8 : 16;      // values a thread
    int log_lanes = 0;
    while ((each << log_lanes) < p.head_dim) ++log_lanes;
    StoreArgs a{{k_packed, v_packed}, {k_rows, v_rows}, {(uint8_t*)p.k_codes, (uint8_t*)p.v_codes}, {(uint8_t*)p.k_scale, (uint8_t*)p.v_scale},
                positions, token_slot, {p.page_table, p.slots, p.table_stride, p.pages}, p.kv_heads, p.head_dim, (unsigned)(T * p.kv_heads), error};
    const unsigned per_block = (kThreads >> log_lanes) * kStoreRows;
    const dim3 grid((a.rows_of_each + per_block - 1) / per_block, 2);
    const unsigned per_kv_head = p.kv_heads == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / (unsigned)p.kv_heads);
    note_launch();
    auto launch = [&](auto kernel) {
        launch_kernel("kv_quant_store", kernel, grid, dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a, log_lanes, per_kv_head);
    };
    auto of_type = [&](auto fp8, auto int8) { p.fmt == QUANT_FP8 ? launch(fp8) : launch(int8); };
    if (dt == F32) of_type(kv_quant_store_kernel<float, QUANT_FP8, 8>, kv_quant_store_kernel<float, QUANT_INT8, 8>);
    else if (each == 16) of_type(kv_quant_store_kernel<__nv_bfloat16, QUANT_FP8, 16>, kv_quant_store_kernel<__nv_bfloat16, QUANT_INT8, 16>);
    else of_type(kv_quant_store_kernel<__nv_bfloat16, QUANT_FP8, 8>, kv_quant_store_kernel<__nv_bfloat16, QUANT_INT8, 8>);
}

void kv_quant_load(const QuantPools& p, DType dt, int n_seqs, const int32_t* slot_ids, const int32_t* seq_ends, void* k_out, void* v_out,
                   int32_t* out_table, int pages, bool whole, long long room, int read_seqs, int read_pages, const int32_t* cu_seqlens,
                   int skip_new, bool attend, int window, int* error, cudaStream_t stream) {
    if (whole) { read_seqs = n_seqs; read_pages = pages; }
    if (n_seqs <= 0 || pages <= 0 || read_seqs <= 0 || read_pages <= 0) return;
    check_pools("kv_quant_load", p);
    if (read_seqs > 65535) throw std::invalid_argument("kv_quant_load: more than 65535 sequences");
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) throw std::invalid_argument("kv_quant_load: outputs must be 16-byte aligned");
    if (whole && !out_table) throw std::invalid_argument("kv_quant_load: the pages of whole sequences need a page table");
    if (room > 0x7fffffffll) throw std::invalid_argument("kv_quant_load: more than 2^31 pages in one call");
    LoadArgs a{{(const uint8_t*)p.k_codes, (const uint8_t*)p.v_codes}, {(const uint8_t*)p.k_scale, (const uint8_t*)p.v_scale}, {k_out, v_out}, out_table,
               slot_ids, seq_ends, {p.page_table, p.slots, p.table_stride, p.pages}, p.kv_heads, p.head_dim, n_seqs, pages, whole ? 1 : 0, room,
               cu_seqlens, whole ? 0 : skip_new, attend ? 1 : 0, attend ? window : 0, error};
    note_launch();
    auto kernel = dt == F32 ? (p.fmt == QUANT_FP8 ? kv_quant_load_kernel<float, QUANT_FP8> : kv_quant_load_kernel<float, QUANT_INT8>)
                            : (p.fmt == QUANT_FP8 ? kv_quant_load_kernel<__nv_bfloat16, QUANT_FP8> : kv_quant_load_kernel<__nv_bfloat16, QUANT_INT8>);
    launch_kernel("kv_quant_load", kernel, dim3((unsigned)read_pages, (unsigned)read_seqs, 2), dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a);
}

}  // namespace sm
