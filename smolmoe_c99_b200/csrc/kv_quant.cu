// Writing the 8-bit key/value cache and reading it back (the format: kv_quant.cuh).
//
// Both are bound by memory: a thread takes 8 values of a row at a time (16 or 32 bytes in, 8 out, or the other way) and
// several rows at once; the lanes that share a row find its largest magnitude with shuffles, so a value is read once and
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

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
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

// One row per group of `lanes` threads (a power of two, at least head_dim / 8); blockIdx.y: keys or values. A thread does
// kStoreRows rows, so that as many loads are under way together.
constexpr int kStoreRows = 2;

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) kv_quant_store_kernel(StoreArgs a, int lanes) {
    pdl_wait();                  // the rows come from the kernel before
    pdl_launch_dependents();
    const int per_block = kThreads / lanes;
    const unsigned row0 = blockIdx.x * (per_block * kStoreRows) + threadIdx.x / lanes;
    const int part = threadIdx.x % lanes;
    // (chosen, not indexed: an index that is not a constant would put the arguments into local memory)
    const bool keys = blockIdx.y == 0;
    const T* packed = (const T*)(keys ? a.packed[0] : a.packed[1]);
    T* rows = (T*)(keys ? a.rows[0] : a.rows[1]);
    uint8_t* codes = keys ? a.codes[0] : a.codes[1];
    uint8_t* scales = keys ? a.scales[0] : a.scales[1];
    float x[kStoreRows][8];
    int at_token[kStoreRows], at_slot[kStoreRows], kv_head[kStoreRows];
    bool mine[kStoreRows];
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) {
        const unsigned row = row0 + u * per_block;
        const bool live = row < a.rows_of_each;
        mine[u] = live && part * 8 < a.head_dim;
        const unsigned t = live ? row / (unsigned)a.kv_heads : 0;
        kv_head[u] = (int)(row - t * (unsigned)a.kv_heads);
        at_token[u] = a.positions[t];
        at_slot[u] = a.token_slot[t];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
        if (mine[u]) load8(packed + (size_t)row * a.head_dim + part * 8, x[u]);
    }
    int page[kStoreRows];
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) page[u] = at_token[u] < 0 ? -1 : a.pages.at(at_slot[u], at_token[u] / kPageSize);
#pragma unroll
    for (int u = 0; u < kStoreRows; ++u) {
        const unsigned row = row0 + u * per_block;
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[u][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, amax, o);
            if (o < lanes) amax = max(amax, other);
        }
        if (mine[u]) {
            const int byte = scale_byte<FMT>(amax);
            uint32_t lo = 0, hi = 0;
            if (byte != kNoScale) {
                const float up = power_of_two(127 - byte);
                lo = encode4<FMT>(x[u][0] * up, x[u][1] * up, x[u][2] * up, x[u][3] * up);
                hi = encode4<FMT>(x[u][4] * up, x[u][5] * up, x[u][6] * up, x[u][7] * up);
            }
            if (page[u] >= 0) {
                const size_t cell = ((size_t)page[u] * a.kv_heads + kv_head[u]) * kPageSize + at_token[u] % kPageSize;
                *reinterpret_cast<uint2*>(codes + cell * a.head_dim + part * 8) = make_uint2(lo, hi);
                if (part == 0) scales[cell] = (uint8_t)byte;
            } else if (a.error) {
                atomicExch(a.error, kBadPlaceInStore);
            }
            if (rows != nullptr) {
                const float scale = scale_of(byte);
                float v[4], w[4];
                decode4<FMT>(lo, v);
                decode4<FMT>(hi, w);
                const float y[8] = {v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale, w[0] * scale, w[1] * scale, w[2] * scale, w[3] * scale};
                store8(rows + (size_t)row * a.head_dim + part * 8, y);
            }
        }
    }
}

struct LoadArgs {
    const uint8_t* codes[2];
    const uint8_t* scales[2];
    void* out[2];                // [sequences, pages, kv_heads, kPageSize, head_dim]
    int32_t* out_table;          // [slots, pages]: where a slot's pages lie in `out`
    const int32_t* slot_ids;     // [sequences]
    const int32_t* seq_ends;     // [sequences]
    QuantPages table;
    int kv_heads, head_dim, pages, whole;
    const int32_t* cu;           // [sequences + 1] (read only where skip_new or a window asks for it)
    int skip_new;                // sequences that bring at most this many tokens are left out
    int attend, window;          // see kv_quant_load in kernels.h
    int* error;
};

// A CTA reads one page (blockIdx.x) of one sequence (blockIdx.y), keys or values (blockIdx.z): a page's kv heads lie one
// behind the other in the pools and in the output, so this is one run of bytes and one of values, 8 of them a thread and
// kLoadSteps such pieces under way together. Positions at and past the sequence's end read as zero; pages wholly past it
// are left alone unless `whole`.
constexpr int kLoadSteps = 4;

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) kv_quant_load_kernel(LoadArgs a) {
    pdl_wait();                  // the cache may have been written by the kernel before
    pdl_launch_dependents();
    const int page = blockIdx.x, seq = blockIdx.y, which = blockIdx.z;
    const int slot = a.slot_ids[seq], end = a.seq_ends[seq];
    if (a.skip_new > 0 && a.cu[seq + 1] - a.cu[seq] <= a.skip_new) return;
    if ((unsigned)slot >= (unsigned)a.table.slots) {
        if (a.error && threadIdx.x == 0) atomicExch(a.error, kBadPlaceInLoad);
        return;
    }
    if (which == 0 && threadIdx.x == 0) a.out_table[(size_t)slot * a.pages + page] = seq * a.pages + page;
    const int live = min(end - page * kPageSize, kPageSize);      // positions of the page that the sequence holds
    if (live <= 0 && !a.whole) return;
    if (a.window > 0) {
        // pages that no token of the step sees, but for the neighbour that shares a tile of 128 positions with a seen one
        const int lowest = end - (a.cu[seq + 1] - a.cu[seq]) - a.window + 1;
        if (lowest > 0 && page < lowest / 128 * (128 / kPageSize)) return;
    }
    const int held = live > 0 ? a.table.at(slot, page) : -1;
    if (live > 0 && held < 0 && a.error && threadIdx.x == 0) atomicExch(a.error, kBadPlaceInLoad);
    const int parts = a.head_dim / 8, total = a.kv_heads * kPageSize * parts;      // pieces of 8 values: of a row, of the page
    const size_t cell0 = held < 0 ? 0 : (size_t)held * a.kv_heads * kPageSize;
    const uint8_t* codes = a.codes[which] + cell0 * a.head_dim;
    T* out = (T*)a.out[which] + ((size_t)seq * a.pages + page) * a.kv_heads * kPageSize * a.head_dim;
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
    int lanes = 1;
    while (lanes * 8 < p.head_dim) lanes *= 2;
    StoreArgs a{{k_packed, v_packed}, {k_rows, v_rows}, {(uint8_t*)p.k_codes, (uint8_t*)p.v_codes}, {(uint8_t*)p.k_scale, (uint8_t*)p.v_scale},
                positions, token_slot, {p.page_table, p.slots, p.table_stride, p.pages}, p.kv_heads, p.head_dim, (unsigned)(T * p.kv_heads), error};
    const unsigned per_block = kThreads / lanes * kStoreRows;
    const dim3 grid((a.rows_of_each + per_block - 1) / per_block, 2);
    note_launch();
    auto kernel = dt == F32 ? (p.fmt == QUANT_FP8 ? kv_quant_store_kernel<float, QUANT_FP8> : kv_quant_store_kernel<float, QUANT_INT8>)
                            : (p.fmt == QUANT_FP8 ? kv_quant_store_kernel<__nv_bfloat16, QUANT_FP8> : kv_quant_store_kernel<__nv_bfloat16, QUANT_INT8>);
    launch_kernel("kv_quant_store", kernel, grid, dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a, lanes);
}

void kv_quant_load(const QuantPools& p, DType dt, int n_seqs, const int32_t* slot_ids, const int32_t* seq_ends, void* k_out, void* v_out,
                   int32_t* out_table, int pages, bool whole, const int32_t* cu_seqlens, int skip_new, bool attend, int window,
                   int* error, cudaStream_t stream) {
    if (n_seqs <= 0 || pages <= 0) return;
    check_pools("kv_quant_load", p);
    if (n_seqs > 65535) throw std::invalid_argument("kv_quant_load: more than 65535 sequences");
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) throw std::invalid_argument("kv_quant_load: outputs must be 16-byte aligned");
    LoadArgs a{{(const uint8_t*)p.k_codes, (const uint8_t*)p.v_codes}, {(const uint8_t*)p.k_scale, (const uint8_t*)p.v_scale}, {k_out, v_out}, out_table,
               slot_ids, seq_ends, {p.page_table, p.slots, p.table_stride, p.pages}, p.kv_heads, p.head_dim, pages, whole ? 1 : 0, cu_seqlens, skip_new,
               attend ? 1 : 0, attend ? window : 0, error};
    note_launch();
    auto kernel = dt == F32 ? (p.fmt == QUANT_FP8 ? kv_quant_load_kernel<float, QUANT_FP8> : kv_quant_load_kernel<float, QUANT_INT8>)
                            : (p.fmt == QUANT_FP8 ? kv_quant_load_kernel<__nv_bfloat16, QUANT_FP8> : kv_quant_load_kernel<__nv_bfloat16, QUANT_INT8>);
    launch_kernel("kv_quant_load", kernel, dim3((unsigned)pages, (unsigned)n_seqs, 2), dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a);
}

}  // namespace sm
