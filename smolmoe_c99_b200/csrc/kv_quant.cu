// Writing the 8-bit key/value cache and reading it back (the format: kv_quant.cuh).
//
// Both are bound by memory: a thread takes 8 values of a row (16 or 32 bytes in, 8 out, or the other way), the lanes that
// share a row find its largest magnitude with shuffles, so a value is read once and written once.
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
    long long rows_of_each;      // T * kv_heads
    int* error;
};

// One row per group of `lanes` threads (a power of two, at least head_dim / 8); blockIdx.y: keys or values.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) kv_quant_store_kernel(StoreArgs a, int lanes) {
    pdl_wait();                  // the rows come from the kernel before
    pdl_launch_dependents();
    const int per_block = kThreads / lanes;
    const long long row = (long long)blockIdx.x * per_block + threadIdx.x / lanes;
    const int part = threadIdx.x % lanes;
    const int which = blockIdx.y;
    const bool live = row < a.rows_of_each, mine = live && part * 8 < a.head_dim;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const size_t at = (size_t)row * a.head_dim + part * 8;
    size_t cell = 0;             // the row's number in the pools
    bool placed = true;
    if (live) {
        const int t = (int)(row / a.kv_heads), kvh = (int)(row - (long long)t * a.kv_heads);
        const int pos = a.positions[t];
        const int page = pos < 0 ? -1 : a.pages.at(a.token_slot[t], pos / kPageSize);
        if (page < 0) {
            if (a.error) atomicExch(a.error, kBadPlaceInStore);
            placed = false;
        }
        cell = ((size_t)page * a.kv_heads + kvh) * kPageSize + pos % kPageSize;
    }
    if (mine) load8((const T*)a.packed[which] + at, x);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
    for (int o = lanes >> 1; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!mine) return;
    const int byte = scale_byte<FMT>(amax);
    uint32_t lo = 0, hi = 0;
    if (byte != kNoScale) {
        const float up = power_of_two(127 - byte);
        lo = encode4<FMT>(x[0] * up, x[1] * up, x[2] * up, x[3] * up);
        hi = encode4<FMT>(x[4] * up, x[5] * up, x[6] * up, x[7] * up);
    }
    if (placed) {
        *reinterpret_cast<uint2*>(a.codes[which] + cell * a.head_dim + part * 8) = make_uint2(lo, hi);
        if (part == 0) a.scales[which][cell] = (uint8_t)byte;
    }
    if (a.rows[which] != nullptr) {
        const float scale = scale_of(byte);
        float v[4], w[4];
        decode4<FMT>(lo, v);
        decode4<FMT>(hi, w);
        const float y[8] = {v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale, w[0] * scale, w[1] * scale, w[2] * scale, w[3] * scale};
        store8((T*)a.rows[which] + at, y);
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

// blockIdx.y: the sequence, blockIdx.z: keys or values; a thread takes 8 values. Positions at and past the sequence's end
// read as zero; pages wholly past it are left alone unless `whole`.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) kv_quant_load_kernel(LoadArgs a) {
    pdl_wait();                  // the cache may have been written by the kernel before
    pdl_launch_dependents();
    const int seq = blockIdx.y, which = blockIdx.z;
    const int slot = a.slot_ids[seq], end = a.seq_ends[seq];
    if (a.skip_new > 0 && a.cu[seq + 1] - a.cu[seq] <= a.skip_new) return;
    const int parts = a.head_dim / 8;                             // of a row
    const long long idx = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int part = (int)(idx % parts);
    const long long row = idx / parts;                            // page, kv head, position in the page
    const int in_page = (int)(row % kPageSize);
    const int kvh = (int)((row / kPageSize) % a.kv_heads);
    const int page = (int)(row / ((long long)kPageSize * a.kv_heads));
    if (page >= a.pages) return;
    if ((unsigned)slot >= (unsigned)a.table.slots) {
        if (a.error) atomicExch(a.error, kBadPlaceInLoad);
        return;
    }
    if (which == 0 && part == 0 && in_page == 0 && kvh == 0) a.out_table[(size_t)slot * a.pages + page] = seq * a.pages + page;
    if (page * kPageSize >= end && !a.whole) return;
    if (a.window > 0) {
        // pages that no token of the step sees, but for the neighbour that shares a tile of 128 positions with a seen one
        const int lowest = end - (a.cu[seq + 1] - a.cu[seq]) - a.window + 1;
        if (lowest > 0 && page < lowest / 128 * (128 / kPageSize)) return;
    }
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int held = page * kPageSize + in_page < end ? a.table.at(slot, page) : -1;
    if (held < 0) {
        if (page * kPageSize + in_page < end && a.error) atomicExch(a.error, kBadPlaceInLoad);
    } else {
        const size_t cell = ((size_t)held * a.kv_heads + kvh) * kPageSize + in_page;
        int byte = a.scales[which][cell];
        if (a.attend) {
            if (which == 0 && a.scales[1][cell] == kNoScale) byte = kNoScale;
            if (which == 1 && byte == kNoScale) byte = 0;
        }
        const float scale = scale_of(byte);
        const uint2 codes = *reinterpret_cast<const uint2*>(a.codes[which] + cell * a.head_dim + part * 8);
        float v[4], w[4];
        decode4<FMT>(codes.x, v);
        decode4<FMT>(codes.y, w);
        const bool none = byte == kNoScale;      // (also where the codes are another row's: a key whose value has no scale)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = none ? __int_as_float(0x7fffffff) : v[i] * scale;
            y[4 + i] = none ? __int_as_float(0x7fffffff) : w[i] * scale;
        }
    }
    const size_t out_row = (size_t)seq * a.pages * a.kv_heads * kPageSize + (size_t)row;
    store8((T*)a.out[which] + out_row * a.head_dim + part * 8, y);
}

void check_sizes(const char* who, int kv_heads, int head_dim, int fmt) {
    if (kv_heads <= 0 || head_dim <= 0 || head_dim % 8 || head_dim > 256)
        throw std::invalid_argument(std::string(who) + ": head_dim " + std::to_string(head_dim) + " is not a multiple of 8 up to 256");
    if (fmt != QUANT_FP8 && fmt != QUANT_INT8) throw std::invalid_argument(std::string(who) + ": unknown format " + std::to_string(fmt));
}

}  // namespace

void kv_quant_store(const void* k_packed, const void* v_packed, DType dt, int T, int kv_heads, int head_dim, void* k_rows,
                    void* v_rows, int fmt, void* k_pool, void* v_pool, void* k_scale, void* v_scale, long long pool_pages,
                    const int32_t* positions, const int32_t* page_table, int slots, int table_stride, const int32_t* token_slot, cudaStream_t stream) {
    if (T <= 0) return;
    check_sizes("kv_quant_store", kv_heads, head_dim, fmt);
    if (((uintptr_t)k_packed | (uintptr_t)v_packed | (uintptr_t)k_rows | (uintptr_t)v_rows) & 15 || ((uintptr_t)k_pool | (uintptr_t)v_pool) & 7)
        throw std::invalid_argument("kv_quant_store: rows must be 16-byte aligned and pools 8-byte aligned");
    int lanes = 1;
    while (lanes * 8 < head_dim) lanes *= 2;
    StoreArgs a{{k_packed, v_packed}, {k_rows, v_rows}, {(uint8_t*)k_pool, (uint8_t*)v_pool}, {(uint8_t*)k_scale, (uint8_t*)v_scale},
                positions, token_slot, {page_table, slots, table_stride, pool_pages}, kv_heads, head_dim, (long long)T * kv_heads, error_word()};
    const long long per_block = kThreads / lanes;
    const dim3 grid((unsigned)((a.rows_of_each + per_block - 1) / per_block), 2);
    note_launch();
    auto kernel = dt == F32 ? (fmt == QUANT_FP8 ? kv_quant_store_kernel<float, QUANT_FP8> : kv_quant_store_kernel<float, QUANT_INT8>)
                            : (fmt == QUANT_FP8 ? kv_quant_store_kernel<__nv_bfloat16, QUANT_FP8> : kv_quant_store_kernel<__nv_bfloat16, QUANT_INT8>);
    launch_kernel("kv_quant_store", kernel, grid, dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a, lanes);
}

void kv_quant_load(int fmt, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                   long long pool_pages, DType dt, int n_seqs, int kv_heads, int head_dim, const int32_t* slot_ids, const int32_t* seq_ends,
                   const int32_t* page_table, int slots, int table_stride, void* k_out, void* v_out, int32_t* out_table, int pages, bool whole,
                   const int32_t* cu_seqlens, int skip_new, bool attend, int window, cudaStream_t stream) {
    if (n_seqs <= 0 || pages <= 0) return;
    check_sizes("kv_quant_load", kv_heads, head_dim, fmt);
    if (n_seqs > 65535) throw std::invalid_argument("kv_quant_load: more than 65535 sequences");
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15 || ((uintptr_t)k_pool | (uintptr_t)v_pool) & 7)
        throw std::invalid_argument("kv_quant_load: outputs must be 16-byte aligned and pools 8-byte aligned");
    LoadArgs a{{(const uint8_t*)k_pool, (const uint8_t*)v_pool}, {(const uint8_t*)k_scale, (const uint8_t*)v_scale}, {k_out, v_out}, out_table,
               slot_ids, seq_ends, {page_table, slots, table_stride, pool_pages}, kv_heads, head_dim, pages, whole ? 1 : 0, cu_seqlens, skip_new, attend ? 1 : 0, attend ? window : 0, error_word()};
    const long long threads = (long long)pages * kv_heads * kPageSize * (head_dim / 8);
    const long long blocks = (threads + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffll) throw std::invalid_argument("kv_quant_load: too many pages for one call");
    note_launch();
    auto kernel = dt == F32 ? (fmt == QUANT_FP8 ? kv_quant_load_kernel<float, QUANT_FP8> : kv_quant_load_kernel<float, QUANT_INT8>)
                            : (fmt == QUANT_FP8 ? kv_quant_load_kernel<__nv_bfloat16, QUANT_FP8> : kv_quant_load_kernel<__nv_bfloat16, QUANT_INT8>);
    launch_kernel("kv_quant_load", kernel, dim3((unsigned)blocks, (unsigned)n_seqs, 2), dim3(kThreads), 0, stream, 1, dependent_launch_enabled(), a);
}

}  // namespace sm
