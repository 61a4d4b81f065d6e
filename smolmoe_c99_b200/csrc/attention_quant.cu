// Attention over the paged 8-bit cache (kv_quant.cuh) for one or a few new tokens per sequence, bfloat16 queries.
//
// What bounds it: reading the cache. So the unit of work is a tile of kTile positions of one kv head, all tiles of all
// sequences (and, for more rows than a tile of the tensor cores takes, all blocks of rows) are put in one line, and every
// CTA of a grid that fills the GPU once takes an equal run of that line, whatever the sequences' lengths are. A run that
// begins or ends inside a sequence leaves the running maximum, the sum and the weighted values of its part in a workspace,
// and a second kernel puts the parts together in the order of the line. (`direct`: few tiles a sequence: a CTA takes one
// whole sequence and kv head, and there is nothing to put together.) All the line needs of the step (lengths, slots,
// pages) is read on the device, so a captured launch follows a growing sequence.
//
// A CTA is eight warps; warp w takes the tiles w, w + 8, ... of the run, each warp with a ring of its own in shared memory
// that the TMA engine fills (codes of 64 or 128 bytes a row as boxes of a tensor map, swizzled so that ldmatrix meets no
// bank conflict; other head sizes as one contiguous copy). Rows of queries are (token, head of the group) and are the
// columns of the products: S^T = K Q^T and O^T = V^T P^T, mma.sync m16n8k16 with positions, and dimensions, as the 16 rows.
// Codes become half-precision operands in registers (exact; two codes an instruction for e4m3). Their fragments come from
//   K: ldmatrix of 16-bit elements: a thread gets four neighbouring codes of its row, which serve as the four elements of a
//      step of 16 dimensions (the order of dimensions in a sum is free: the queries are laid out to match);
//   V: ldmatrix of 8-bit 16 x 16 blocks, transposed: four neighbouring rows (positions) of one dimension.
// The rows that a matrix names are permuted by kRowOf so that both kinds of read are free of bank conflicts and P needs
// no exchange beyond movmatrix.
// Scales: the exponent of a key's row multiplies its scores; that of a value's row goes into the weight. Weights are half
// precision: P * 2^(e - E + 15) with E the largest exponent so far, so the largest weight is 2^15 and what is lost lies 2^40
// below it. The rows of queries are scaled by powers of two to half precision, which holds all 8 bits of a bfloat16.
// Sums, maxima and accumulators are float.
#include <math_constants.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "drain.cuh"
#include "kernels.h"
#include "kv_quant.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace sm {

namespace {

using namespace tc5;

constexpr int kTile = 32;                // positions
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kWaitCode = 34;            // error word: a wait ran out
constexpr int kMaxSeqs = 4096;

struct AttnArgs {
    const __nv_bfloat16* q;              // [T, heads, head_dim]
    __nv_bfloat16* out;
    const uint8_t *k_codes, *v_codes, *k_scale, *v_scale;
    QuantPages pages;
    const int32_t* slot_ids;             // [seqs]
    const int32_t* seq_ends;             // [seqs] lengths after the step
    const int32_t* cu;                   // [seqs + 1] first token of a sequence among the step's
    int seqs, heads, kv_heads, head_dim, window;
    int most_new;                        // sequences with more new tokens are not this kernel's
    int block_tokens;                    // tokens of a block of rows
    int direct, stages;
    float scale_log2;
    float* parts;                        // [CTAs][2][rows][padded head size + 4]: values, then maximum and sum
    int* error;
};

// A sequence's share of the line.
struct Seq {
    int start, n, blocks, first_tile, tiles;   // tiles of one kv head and block of rows
};
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int i) {
    Seq s;
    s.n = a.cu[i + 1] - a.cu[i];
    const int end = a.seq_ends[i];
    s.start = end - s.n;
    s.blocks = s.n <= 0 || s.n > a.most_new || s.start < 0 ? 0 : (s.n + a.block_tokens - 1) / a.block_tokens;
    const int lowest = a.window > 0 ? max(0, s.start - a.window + 1) : 0;
    s.first_tile = lowest / kTile;
    s.tiles = (end - 1) / kTile - s.first_tile + 1;
    return s;
}

// Prefix sums over the sequences, in shared memory: tiles and pairs (kv head, block of rows) before each.
__device__ void scan_sequences(const AttnArgs& a, int* tiles_before, int* pairs_before) {
    __shared__ int2 warp_total[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 carry = make_int2(0, 0);
    for (int base = 0; base < a.seqs; base += kThreads) {
        const int i = base + threadIdx.x;
        int2 mine = make_int2(0, 0);
        if (i < a.seqs) {
            const Seq s = seq_of(a, i);
            mine.y = a.kv_heads * s.blocks;
            mine.x = mine.y * s.tiles;
        }
        int2 run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, run.x, o), y = __shfl_up_sync(0xffffffffu, run.y, o);
            if (lane >= o) { run.x += x; run.y += y; }
        }
        if (lane == 31) warp_total[warp] = run;
        __syncthreads();
        int2 before = carry;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int2 t = warp_total[w];
            if (w < warp) { before.x += t.x; before.y += t.y; }
            carry.x += t.x;
            carry.y += t.y;
        }
        if (i < a.seqs) {
            tiles_before[i] = before.x + run.x - mine.x;
            pairs_before[i] = before.y + run.y - mine.y;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) { tiles_before[a.seqs] = carry.x; pairs_before[a.seqs] = carry.y; }
    __syncthreads();
}
// The last i with before[i] <= x (x below before[seqs]: then before[i + 1] > x).
__device__ __forceinline__ int find_seq(const int* before, int seqs, int x) {
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}
// Tiles of the line that a CTA takes: at least one for each warp.
__device__ __forceinline__ int run_of(int total, int ctas) { return max((total + ctas - 1) / ctas, kWarps); }

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Two 16 x 16 blocks of bytes (lanes 0-15 name the rows of the first, 16-31 of the second), transposed: a thread gets, of
// block i, rows 4 * (lane % 4) .. + 3 of column lane / 4 in r[2 i] and of column lane / 4 + 8 in r[2 i + 1].
__device__ __forceinline__ void ldmatrix_bytes_trans_x2(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Row r (0..15) of a block of 16 positions, as the tensor-core tile numbers them, is this position of the block: distinct
// modulo 8 among the rows that one ldmatrix phase reads, for the keys (rows 0-7, 8-15) and for the values (rows 0, 1, 8, 9,
// 2, 3, 10, 11, and the other eight).
__device__ __forceinline__ int row_position(int r) { return r < 8 ? r : 8 + ((r - 8) ^ 4); }

// NB: blocks of 64 of the head dimension. NHT: tiles of 8 rows of queries. BOX: head_dim is 64 * NB.
template <int NB, int NHT, int FMT, bool BOX>
__global__ void __launch_bounds__(kThreads, 1) attention_quant_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v, AttnArgs a) {
    constexpr int HDP = NB * 64, LD = HDP + 4;      // padded head size; a row of the warps' results (conflict-free)
    constexpr int CH = HDP / 16;                    // pieces of 16 dimensions
    constexpr int R = 8 * NHT;                      // rows of queries
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int hd = BOX ? HDP : a.head_dim, group = a.heads / a.kv_heads;
    const int pieces = BOX ? CH : hd / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    const int tile_bytes = kTile * hd;              // of keys; as many of values
    const int slot_bytes = 2 * tile_bytes;
    const int S = a.stages;
    unsigned char* ring0 = BOX ? reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) : smem_raw;
    unsigned char* ring = ring0 + (size_t)warp * S * slot_bytes;
    float* wo = reinterpret_cast<float*>(ring0 + (size_t)kWarps * S * slot_bytes);   // [warp][R][LD]
    float* wm = wo + kWarps * R * LD;               // [warp][R] maxima, then the warps' factors
    float* wl = wm + kWarps * R;                    // [warp][R] sums
    float* row_m = wl + kWarps * R;                 // [R]
    float* row_l = row_m + R;                       // [R]
    unsigned char* scales = reinterpret_cast<unsigned char*>(row_l + R) + (size_t)warp * S * 2 * kTile;   // [warp][stage][exponents of keys, values]
    uint64_t* bars0 = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(row_l + R) + (size_t)kWarps * S * 2 * kTile);
    uint64_t* bars = bars0 + warp * S;              // [warp][stage]
    int* tiles_before = reinterpret_cast<int*>(bars0 + kWarps * S);                  // [seqs + 1]
    int* pairs_before = tiles_before + a.seqs + 1;                                   // [seqs + 1]

    if (lane == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&bars[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                  // q and the cache come from the kernels before
    pdl_launch_dependents();
    scan_sequences(a, tiles_before, pairs_before);

    int u_lo, u_hi, run = 0;
    if (a.direct) {
        if ((int)blockIdx.x >= pairs_before[a.seqs]) return;
        const int i = find_seq(pairs_before, a.seqs, blockIdx.x);
        const int tiles = seq_of(a, i).tiles;
        u_lo = tiles_before[i] + ((int)blockIdx.x - pairs_before[i]) * tiles;
        u_hi = u_lo + tiles;
    } else {
        const int total = tiles_before[a.seqs];
        run = run_of(total, gridDim.x);
        u_lo = min(total, (int)blockIdx.x * run);
        u_hi = min(total, u_lo + run);
    }
    const int my_tiles = u_hi - u_lo > warp ? (u_hi - u_lo - warp + kWarps - 1) / kWarps : 0;

    // Where this warp's tiles 32 * batch + lane lie: the row of the pools (pages of kv heads of 64 positions) of its first
    // position. 32 are looked up at once, a lane each.
    auto locate = [&](int batch) -> int {
        const int k = batch * 32 + lane;
        if (k >= my_tiles) return 0;
        const int u = u_lo + warp + kWarps * k;
        const int i = find_seq(tiles_before, a.seqs, u);
        const Seq s = seq_of(a, i);
        const int pair = (u - tiles_before[i]) / s.tiles, t = u - tiles_before[i] - pair * s.tiles;
        const int key = (s.first_tile + t) * kTile;
        int page = a.pages.at(a.slot_ids[i], key / kPageSize);
        if (page < 0) {
            if (a.error) atomicExch(a.error, kBadPlaceInAttention);
            page = 0;
        }
        return (page * a.kv_heads + pair / s.blocks) * kPageSize + key % kPageSize;
    };
    int places = locate(0), place_batch = 0;
    // Asks for this warp's tile k into its stage of the ring (all lanes call it, in order of k).
    auto request = [&](int k, int stage) {
        if ((k >> 5) != place_batch) {
            place_batch = k >> 5;
            places = locate(place_batch);
        }
        const int row = __shfl_sync(0xffffffffu, places, k & 31);
        unsigned char* slot = ring + (size_t)stage * slot_bytes;
        uint64_t* bar = &bars[stage];
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(2 * tile_bytes + 2 * kTile));
        __syncwarp();
        if (lane < 2) {
            unsigned char* dst = slot + lane * tile_bytes;
            if (BOX) tma_load_2d(dst, lane ? &map_v : &map_k, 0, row, bar);
            else bulk_load(dst, (lane ? a.v_codes : a.k_codes) + (size_t)row * hd, (uint32_t)tile_bytes, bar);
        } else if (lane < 4) {
            bulk_load(scales + (stage * 2 + lane - 2) * kTile, (lane == 3 ? a.v_scale : a.k_scale) + row, kTile, bar);
        }
    };
    const int ahead = min(S, my_tiles);
    for (int k = 0; k < ahead; ++k) request(k, k);
    int issued = ahead, waited = 0, stage = 0;
    uint32_t parity = 0;
    bool ok = true;

    // Shared-memory addresses of the fragments: the row this lane names in an ldmatrix, and its piece of 16 bytes
    auto piece_at = [&](int row, int piece) -> uint32_t {
        if (BOX && NB == 2) return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
        if (BOX) return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
        return (uint32_t)(row * hd + (piece << 4));
    };
    const int k_row = row_position((lane & 7) + ((lane >> 3) & 1) * 8), k_piece = lane >> 4;
    const int v_at = lane & 15;     // the row of the 16 x 16 block this lane names: position of tile row 2 (at / 4) + (at & 1) + 8 (at / 2 & 1)
    const int v_row = row_position(2 * (v_at >> 2) + (v_at & 1) + ((v_at >> 1) & 1) * 8), v_piece = lane >> 4;
    const int pos_lo = g, pos_hi = 8 + (g ^ 4);      // positions of a block of 16 whose scores this thread holds

    int k = 0;
    for (int u = u_lo; u < u_hi;) {
        // ---- one part of one sequence, kv head and block of rows -------------------------------------------------
        const int i = find_seq(tiles_before, a.seqs, u);
        const Seq s = seq_of(a, i);
        const int pair = (u - tiles_before[i]) / s.tiles;
        const int pair_at = tiles_before[i] + pair * s.tiles, part_end = min(u_hi, pair_at + s.tiles);
        const int kvh = pair / s.blocks, block = pair - kvh * s.blocks;
        const int token0 = block * a.block_tokens, tokens = min(a.block_tokens, s.n - token0), rows = tokens * group;
        const int first_pos = s.start + token0, last_pos = first_pos + tokens - 1;
        const int lowest = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
        const size_t q_row0 = (size_t)(a.cu[i] + token0) * a.heads + (size_t)kvh * group;    // row r: + (r / group) * heads + r % group

        // the rows of queries as half precision, scaled by a power of two to at most 2^11
        uint32_t qf[CH][NHT][2];
        float q_scale[NHT][2];           // of rows 2 q4 and 2 q4 + 1 of a tile: undoes the power of two, times scale * log2(e)
        int row_pos[NHT][2];             // their positions
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh) {
            const int r = nh * 8 + g;
            const __nv_bfloat16* src = a.q + (q_row0 + (size_t)(r / group) * a.heads + r % group) * hd;
            uint2 raw[CH];
            uint32_t amax = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                raw[c] = make_uint2(0, 0);
                if (r < rows && (BOX || c < pieces)) raw[c] = *reinterpret_cast<const uint2*>(src + c * 16 + q4 * 4);
                const uint32_t m0 = raw[c].x & 0x7fff7fffu, m1 = raw[c].y & 0x7fff7fffu;
                amax = max(amax, max(max(m0 & 0xffffu, m0 >> 16), max(m1 & 0xffffu, m1 >> 16)));
            }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // exponent of the largest magnitude; rows with an infinity or a NaN keep their values (and their results are NaN)
            const int E = amax >= 0x7f80u ? 10 : max((int)(amax >> 7) - 127, -110);
            const float up = power_of_two(10 - E);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                qf[c][nh][0] = pack_half2(__uint_as_float(raw[c].x << 16) * up, __uint_as_float(raw[c].x & 0xffff0000u) * up);
                qf[c][nh][1] = pack_half2(__uint_as_float(raw[c].y << 16) * up, __uint_as_float(raw[c].y & 0xffff0000u) * up);
            }
            const float down = power_of_two(E - 10) * a.scale_log2;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                q_scale[nh][e] = __shfl_sync(0xffffffffu, down, (2 * q4 + e) * 4);
                row_pos[nh][e] = first_pos + min((nh * 8 + 2 * q4 + e) / group, tokens - 1);
            }
        }
        float ot[CH][NHT][4];
        float run_m[NHT][2], run_l[NHT][2];
        int top_exponent = 0;            // E, as a byte; 0: none yet
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh) {
            run_m[nh][0] = run_m[nh][1] = -CUDART_INF_F;
            run_l[nh][0] = run_l[nh][1] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) ot[c][nh][0] = ot[c][nh][1] = ot[c][nh][2] = ot[c][nh][3] = 0.f;
        }

        for (; k < my_tiles && u_lo + warp + kWarps * k < part_end && ok; ++k) {
            const int key0 = (s.first_tile + (u_lo + warp + kWarps * k - pair_at)) * kTile;
            unsigned char* slot = ring + (size_t)stage * slot_bytes;
            if (!__all_sync(0xffffffffu, mbar_wait(&bars[stage], parity))) {
                if (lane == 0 && a.error) atomicExch(a.error, kWaitCode);
                ok = false;
                break;
            }
            waited = k + 1;
            const uint32_t kt = smem_u32(slot), vt = kt + (uint32_t)tile_bytes;
            const uint8_t* ks = scales + stage * 2 * kTile;
            const uint8_t* vs = ks + kTile;
            // every row sees every position of the tile, or a mask is needed
            const bool masked = key0 + kTile - 1 > first_pos || (a.window > 0 && key0 <= last_pos - a.window);
            int top = vs[lane];
            if (masked) {
                const int from = max(lowest - key0, 0), to = last_pos + 1 - key0;    // positions some row sees: [from, to)
                if (lane < from || lane >= to) top = 0;
                if (from > 0 || to < kTile) {
                    // value rows that no row sees may hold bytes that were never written: zeros (times zero weights)
                    for (int idx = lane; idx < kTile * pieces; idx += 32) {
                        const int row = idx / pieces, piece = idx - row * pieces;
                        if (row < from || row >= to) *reinterpret_cast<uint4*>(slot + tile_bytes + piece_at(row, piece)) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
            }
            if (top == kNoScale) top = 0;
            top = (int)__reduce_max_sync(0xffffffffu, (unsigned)top);
            // S^T = K Q^T
            float st[2][NHT][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int nh = 0; nh < NHT; ++nh) st[mt][nh][0] = st[mt][nh][1] = st[mt][nh][2] = st[mt][nh][3] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                if (!BOX && c >= pieces) break;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    uint32_t w[4];       // rows 0-7 and 8-15 of piece c, then of piece c + 1 (an odd last piece is read twice)
                    const int piece = BOX ? c + k_piece : min(c + k_piece, pieces - 1);
                    ldmatrix_x4(w, kt + piece_at(mt * 16 + k_row, piece));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!BOX && c + half >= pieces) break;
                        uint32_t a0, a1, a2, a3;
                        decode4<FMT>(w[2 * half], a0, a2);
                        decode4<FMT>(w[2 * half + 1], a1, a3);
#pragma unroll
                        for (int nh = 0; nh < NHT; ++nh) mma_f16(st[mt][nh], a0, a1, a2, a3, qf[c + half][nh][0], qf[c + half][nh][1]);
                    }
                }
            }
            // scores (in powers of two), mask, running maxima
            float mx[NHT][2];
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh) { mx[nh][0] = run_m[nh][0]; mx[nh][1] = run_m[nh][1]; }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const float f0 = scale_of(ks[mt * 16 + pos_lo]), f1 = scale_of(ks[mt * 16 + pos_hi]);
#pragma unroll
                for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = st[mt][nh][e] * ((e & 2) ? f1 : f0) * q_scale[nh][e & 1];
                        if (masked) {
                            const int key = key0 + mt * 16 + ((e & 2) ? pos_hi : pos_lo), pos = row_pos[nh][e & 1];
                            if (key > pos || (a.window > 0 && key <= pos - a.window)) x = -CUDART_INF_F;
                        }
                        st[mt][nh][e] = x;
                        mx[nh][e & 1] = fmaxf(mx[nh][e & 1], x);
                    }
            }
            bool moved = top > top_exponent;
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = mx[nh][e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    mx[nh][e] = x;
                    moved |= x > run_m[nh][e];
                }
            if (__any_sync(0xffffffffu, moved)) {
                // a larger maximum or exponent: what has been added up is put on the new footing
                const int drop = max(top - top_exponent, 0);
                const float less = top_exponent == 0 ? 0.f : power_of_two(-min(drop, 126));
                top_exponent = max(top, top_exponent);
#pragma unroll
                for (int nh = 0; nh < NHT; ++nh) {
                    float f[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float by = mx[nh][e] == -CUDART_INF_F ? 1.f : ex2_approx(run_m[nh][e] - mx[nh][e]);
                        run_m[nh][e] = mx[nh][e];
                        run_l[nh][e] *= by;
                        f[e] = by * less;
                    }
#pragma unroll
                    for (int c = 0; c < CH; ++c) { ot[c][nh][0] *= f[0]; ot[c][nh][1] *= f[1]; ot[c][nh][2] *= f[0]; ot[c][nh][3] *= f[1]; }
                }
            }
            // P = 2^(score - maximum), and the weights P * 2^(e - E + 15) as the B operand
            uint32_t pb[2][NHT][2];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int b0 = vs[mt * 16 + pos_lo], b1 = vs[mt * 16 + pos_hi];
                const float w0 = b0 == kNoScale ? CUDART_NAN_F : __int_as_float(max(b0 - top_exponent + 142, 0) << 23);
                const float w1 = b1 == kNoScale ? CUDART_NAN_F : __int_as_float(max(b1 - top_exponent + 142, 0) << 23);
#pragma unroll
                for (int nh = 0; nh < NHT; ++nh) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = st[mt][nh][e];
                        const float ref = run_m[nh][e & 1] == -CUDART_INF_F ? 0.f : run_m[nh][e & 1];
                        const float v = ex2_approx(x - ref);
                        run_l[nh][e & 1] += v;
                        p[e] = masked && x == -CUDART_INF_F ? 0.f : v * ((e & 2) ? w1 : w0);
                    }
                    pb[mt][nh][0] = movmatrix_trans(pack_half2(p[0], p[1]));
                    pb[mt][nh][1] = movmatrix_trans(pack_half2(p[2], p[3]));
                }
            }
            // O^T += V^T P^T
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int c = 0; c < CH; c += 2) {
                    if (!BOX && c >= pieces) break;
                    uint32_t w[4];
                    const int piece = BOX ? c + v_piece : min(c + v_piece, pieces - 1);
                    ldmatrix_bytes_trans_x2(w, vt + piece_at(mt * 16 + v_row, piece));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!BOX && c + half >= pieces) break;
                        uint32_t a0, a1, a2, a3;
                        decode4<FMT>(w[2 * half], a0, a2);
                        decode4<FMT>(w[2 * half + 1], a1, a3);
#pragma unroll
                        for (int nh = 0; nh < NHT; ++nh) mma_f16(ot[c + half][nh], a0, a1, a2, a3, pb[mt][nh][0], pb[mt][nh][1]);
                    }
                }
            __syncwarp();       // every lane has read the slot
            if (k + S < my_tiles) {
                request(k + S, stage);
                issued = k + S + 1;
            }
            if (++stage == S) { stage = 0; parity ^= 1u; }
        }

        // ---- the warps' results put together -------------------------------------------------------------------------
        {
            const float unit = power_of_two(max(top_exponent - 127 - 15, -126));     // (no exponent yet: nothing was added up)
            float* o = wo + (size_t)warp * R * LD;
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float l = run_l[nh][e];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    const int r = nh * 8 + 2 * q4 + e;
                    if (g == 0) { wm[warp * R + r] = run_m[nh][e]; wl[warp * R + r] = l; }
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        o[r * LD + c * 16 + g] = ot[c][nh][e] * unit;
                        o[r * LD + c * 16 + 8 + g] = ot[c][nh][2 + e] * unit;
                    }
                }
        }
        const bool failed = __syncthreads_or(!ok) != 0;
        if (threadIdx.x < R) {
            const int r = threadIdx.x;
            float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, wm[w * R + r]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                // (a warp without positions: 0; without a maximum, because every score it saw is NaN: 1, and its sum is NaN)
                const float f = wm[w * R + r] == -CUDART_INF_F ? (wl[w * R + r] == 0.f ? 0.f : 1.f) : ex2_approx(wm[w * R + r] - m);
                l += wl[w * R + r] * f;
                wm[w * R + r] = f;
            }
            row_m[r] = m;
            row_l[r] = l;
        }
        __syncthreads();
        const bool whole = u == pair_at && part_end == pair_at + s.tiles;
        float* part = a.parts + ((size_t)blockIdx.x * 2 + (pair_at < u_lo ? 0 : 1)) * R * LD;
        for (int idx = threadIdx.x; idx < rows * (HDP / 4); idx += kThreads) {
            const int r = idx / (HDP / 4), d = (idx - r * (HDP / 4)) * 4;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = wm[w * R + r];
                if (f != 0.f) {
                    const float4 x = *reinterpret_cast<const float4*>(wo + ((size_t)w * R + r) * LD + d);
                    sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
                }
            }
            if (failed) continue;
            if (whole) {
                if (BOX || d < hd) {
                    const float inv = 1.0f / row_l[r];
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv), hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
                    *reinterpret_cast<uint2*>(a.out + (q_row0 + (size_t)(r / group) * a.heads + r % group) * hd + d) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                }
            } else {
                *reinterpret_cast<float4*>(part + (size_t)r * LD + d) = sum;
                if (d == 0) { part[(size_t)r * LD + HDP] = row_m[r]; part[(size_t)r * LD + HDP + 1] = row_l[r]; }
            }
        }
        __syncthreads();        // the results' memory is free again
        u = part_end;
    }
    if (!ok) {
        // what was asked for lands before the CTA gives up its shared memory
        OutstandingFill left[8];
        const int n = outstanding_fills(issued, waited, S, left);
        for (int j = 0; j < n; ++j) mbar_wait(&bars[left[j].stage], left[j].parity);
    }
}

// Puts the parts of a (sequence, kv head, block of rows) together, in the order of the line: one CTA per row of queries.
// Threads are (part modulo 8, four dimensions): a thread adds up every eighth part, then the eight sums.
template <int HDP>
__global__ void __launch_bounds__(kThreads) attention_quant_join_kernel(AttnArgs a, int ctas, int rows_of_block) {
    constexpr int LD = HDP + 4, Q = HDP / 4, P = kThreads / 32;      // (a warp holds the dimensions: 16 or 32 lanes of it)
    extern __shared__ int scan[];
    __shared__ float4 sums[P][Q];
    __shared__ float ms[P], ls[P];
    int* tiles_before = scan;
    int* pairs_before = scan + a.seqs + 1;
    // (lengths are no product of the kernel before, which began after what wrote them had ended)
    scan_sequences(a, tiles_before, pairs_before);
    // every CTA waits, those with nothing to do too: this kernel must not end before the one it follows
    pdl_wait();
    pdl_launch_dependents();
    const int pair_at_all = blockIdx.x, r = blockIdx.y, group = a.heads / a.kv_heads;
    if (pair_at_all >= pairs_before[a.seqs]) return;
    const int i = find_seq(pairs_before, a.seqs, pair_at_all);
    const Seq s = seq_of(a, i);
    const int pair = pair_at_all - pairs_before[i], kvh = pair / s.blocks, block = pair - kvh * s.blocks;
    const int token0 = block * a.block_tokens, tokens = min(a.block_tokens, s.n - token0);
    if (r >= tokens * group) return;
    const int run = run_of(tiles_before[a.seqs], ctas);
    const int pair_at = tiles_before[i] + pair * s.tiles;
    const int first = pair_at / run, last = (pair_at + s.tiles - 1) / run;
    if (first == last) return;               // that CTA wrote the row
    const int p = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = first + p; c <= last; c += P) {
        const float* part = a.parts + (((size_t)c * 2 + (pair_at < c * run ? 0 : 1)) * rows_of_block + r) * LD;
        const float pm = part[HDP], pl = part[HDP + 1];
        const float4 x = lane < Q ? *reinterpret_cast<const float4*>(part + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float top = fmaxf(m, pm);
        const float f = m == top || m == -CUDART_INF_F ? 1.f : ex2_approx(m - top), g = pm == top || pm == -CUDART_INF_F ? 1.f : ex2_approx(pm - top);
        m = top;
        l = l * f + pl * g;
        o.x = o.x * f + x.x * g; o.y = o.y * f + x.y * g; o.z = o.z * f + x.z * g; o.w = o.w * f + x.w * g;
    }
    if (lane < Q) sums[p][lane] = o;
    if (lane == 0) { ms[p] = m; ls[p] = l; }
    __syncthreads();
    if (threadIdx.x >= Q) return;
    float top = ms[0];
#pragma unroll
    for (int w = 1; w < P; ++w) top = fmaxf(top, ms[w]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < P; ++w) {
        const float f = ms[w] == -CUDART_INF_F ? 1.f : ex2_approx(ms[w] - top);      // (no maximum: nothing, or NaN)
        const float4 x = sums[w][threadIdx.x];
        total += ls[w] * f;
        sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
    }
    const int d = threadIdx.x * 4;
    if (d >= a.head_dim) return;
    const float inv = 1.0f / total;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv), hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
    const size_t row = (size_t)(a.cu[i] + token0 + r / group) * a.heads + (size_t)kvh * group + r % group;
    *reinterpret_cast<uint2*>(a.out + row * a.head_dim + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

constexpr int kDevices = 64;

int sm_count() {
    static int known[kDevices] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kDevices) return 148;
    if (!known[dev]) cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev);
    return known[dev];
}

template <int NB, int NHT, int FMT, bool BOX>
void launch(AttnArgs a, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, int pairs, int rows_of_block, int most_tiles,
            cudaStream_t stream) {
    constexpr int HDP = NB * 64, R = 8 * NHT;
    const size_t slot = (size_t)2 * kTile * a.head_dim + 2 * kTile;      // codes, and exponents apart from them
    const size_t fixed = (BOX ? 1024 : 0) + ((size_t)kWarps * R * (HDP + 4) + 2 * kWarps * R + 2 * R) * sizeof(float) +
                         (size_t)kWarps * 8 * sizeof(uint64_t) + (size_t)2 * (a.seqs + 1) * sizeof(int);
    // one CTA an SM: as many tiles in flight as fit; a CTA of a single sequence and few tiles asks for no more than those
    const size_t room = 226 * 1024;
    int stages = (int)((room - fixed) / (kWarps * slot));
    stages = std::min(std::max(stages, 1), a.direct ? std::max((most_tiles + kWarps - 1) / kWarps, 1) : 6);
    a.stages = stages;
    const size_t smem = fixed + kWarps * stages * slot;
    auto kernel = attention_quant_kernel<NB, NHT, FMT, BOX>;
    static size_t allowed[kDevices] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kDevices) throw std::runtime_error("attention_quant: more devices than it knows");
    if (allowed[dev] < smem) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
        if (e != cudaSuccess) throw std::runtime_error(std::string("attention_quant: ") + cudaGetErrorString(e));
        allowed[dev] = room;
    }
    note_launch();
    launch_kernel("attention_quant", kernel, dim3((unsigned)ctas), dim3(kThreads), smem, stream, 1, dependent_launch_enabled(), mk, mv, a);
    if (a.direct) return;
    note_launch();
    launch_kernel("attention_quant", attention_quant_join_kernel<HDP>, dim3((unsigned)pairs, (unsigned)rows_of_block), dim3(kThreads),
                  (size_t)2 * (a.seqs + 1) * sizeof(int), stream, 1, dependent_launch_enabled(), a, ctas, R);
}

template <int NB, int NHT, int FMT>
void launch_box(const AttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, int pairs, int rows_of_block, int most_tiles,
                cudaStream_t stream) {
    if (a.head_dim == NB * 64) launch<NB, NHT, FMT, true>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
    else launch<NB, NHT, FMT, false>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
}
template <int FMT>
void launch_fmt(const AttnArgs& a, int row_tiles, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, int pairs, int rows_of_block,
                int most_tiles, cudaStream_t stream) {
    if (a.head_dim <= 64) {
        if (row_tiles == 1) launch_box<1, 1, FMT>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
        else if (row_tiles == 2) launch_box<1, 2, FMT>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
        else launch_box<1, 4, FMT>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
    } else {
        if (row_tiles == 1) launch_box<2, 1, FMT>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
        else launch_box<2, 2, FMT>(a, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
    }
}

}  // namespace

bool attention_quant_supports(int heads, int kv_heads, int head_dim, long long pool_pages) {
    return head_dim % 16 == 0 && head_dim >= 16 && head_dim <= 128 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 &&
           pool_pages > 0 && pool_pages * kv_heads * kPageSize < (1ll << 31);
}

// Floats of workspace that a launch needs (0: none).
long long attention_quant_workspace(int head_dim, int row_tiles, bool direct) {
    return direct ? 0 : (long long)sm_count() * 2 * 8 * row_tiles * ((head_dim <= 64 ? 64 : 128) + 4);
}

void attention_quant(const void* q, void* out, int n_seqs, int heads, int kv_heads, int head_dim, float scale, int window, int fmt,
                     const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale, long long pool_pages,
                     const int32_t* page_table, int slots, int table_stride, const int32_t* slot_ids, const int32_t* seq_ends,
                     const int32_t* cu_seqlens, int max_len, int most_new, int row_tiles, int pairs, bool direct, float* workspace,
                     long long workspace_floats, cudaStream_t stream) {
    if (n_seqs <= 0 || pairs <= 0) return;
    if (!attention_quant_supports(heads, kv_heads, head_dim, pool_pages))
        throw std::invalid_argument("attention_quant: " + std::to_string(heads) + " heads on " + std::to_string(kv_heads) + " of size " +
                                    std::to_string(head_dim) + " (multiples of 16 up to 128, at most 16 heads a kv head), or a pool of 2^31 rows");
    const int group = heads / kv_heads;
    if (n_seqs > kMaxSeqs) throw std::invalid_argument("attention_quant: more than " + std::to_string(kMaxSeqs) + " sequences");
    if ((row_tiles != 1 && row_tiles != 2 && (row_tiles != 4 || head_dim > 64)) || 8 * row_tiles < group)
        throw std::invalid_argument("attention_quant: " + std::to_string(row_tiles) + " tiles of rows");
    if (((uintptr_t)q | (uintptr_t)out) & 15 || ((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15)
        throw std::invalid_argument("attention_quant: operands must be 16-byte aligned");
    if (workspace_floats < attention_quant_workspace(head_dim, row_tiles, direct)) throw std::invalid_argument("attention_quant: the workspace is too small");
    AttnArgs a{(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)k_pool, (const uint8_t*)v_pool, (const uint8_t*)k_scale,
               (const uint8_t*)v_scale, {page_table, slots, table_stride, pool_pages}, slot_ids, seq_ends, cu_seqlens, n_seqs, heads,
               kv_heads, head_dim, window, most_new, 8 * row_tiles / group, direct ? 1 : 0, 0, scale * 1.4426950408889634f, workspace, error_word()};
    CUtensorMap mk{}, mv{};
    if (head_dim == 64 || head_dim == 128) {
        // the pools as rows of codes; a box is a tile of positions of one kv head
        const CUtensorMapSwizzle swizzle = head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
        const uint64_t rows = (uint64_t)pool_pages * kv_heads * kPageSize;
        mk = tiled_map_2d("attention_quant", CU_TENSOR_MAP_DATA_TYPE_UINT8, k_pool, (uint64_t)head_dim, rows, (uint64_t)head_dim, (uint32_t)head_dim,
                          kTile, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        mv = tiled_map_2d("attention_quant", CU_TENSOR_MAP_DATA_TYPE_UINT8, v_pool, (uint64_t)head_dim, rows, (uint64_t)head_dim, (uint32_t)head_dim,
                          kTile, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    const int most_tiles = (max_len + kTile - 1) / kTile + 1;
    const int ctas = direct ? pairs : sm_count(), rows_of_block = a.block_tokens * group;
    if (fmt == QUANT_FP8) launch_fmt<QUANT_FP8>(a, row_tiles, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
    else if (fmt == QUANT_INT8) launch_fmt<QUANT_INT8>(a, row_tiles, mk, mv, ctas, pairs, rows_of_block, most_tiles, stream);
    else throw std::invalid_argument("attention_quant: unknown format " + std::to_string(fmt));
}

}  // namespace sm
