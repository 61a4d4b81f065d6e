// Attention over the paged 8-bit cache (kv_quant.cuh) for one or a few new tokens per sequence, bfloat16 queries.
//
// What bounds it: reading the cache, and for little of it the trips to memory one after the other. The unit of work is a
// tile of 32 or 64 positions of one kv head, worked on by one warp for a block of rows of queries: (token, head of the group). A
// pair is a block of rows and its kv head; its tiles are its sequence's. Two ways of sharing the tiles out:
//  - clusters (little work): the eight warps of each of 1 to 8 CTAs share the tiles of one pair and put their results
//    together through shared memory, the CTAs through the leader's (distributed shared memory). One launch, no workspace.
//  - the line (much work): the tiles of all pairs are put in one line, and every warp of a grid that fills the GPU once takes
//    an equal run of it, whatever the sequences' lengths are. Warps meet nobody. A run that begins or ends inside a pair
//    leaves its rows' references, sums and weighted values of its part in a workspace, and a second kernel puts the
//    parts of each cut pair together in the order of the line.
// All that this needs of the step (lengths, slots, pages) is read on the device, so a captured launch follows a growing
// sequence, and results depend on no order of arrival.
//
// Each warp has a ring of its own in shared memory that the TMA engine fills (codes of 64 or 128 bytes a row as boxes of a
// tensor map, swizzled so that ldmatrix meets no bank conflict; other head sizes as one contiguous copy). Rows of queries
// are the columns of the products: S^T = K Q^T and O^T = V^T P^T, mma.sync m16n8k16 with positions, and dimensions, as the
// 16 rows. Codes become half-precision operands in registers (exact; two codes an instruction for e4m3). Their fragments
// come from
//   K: ldmatrix of 16-bit elements: a thread gets four neighbouring codes of its row, which serve as the four elements of a
//      step of 16 dimensions (the order of dimensions in a sum is free: the queries are laid out to match);
//   V: ldmatrix of 8-bit 16 x 16 blocks, transposed: four neighbouring rows (positions) of one dimension.
// The rows that a matrix names are permuted by row_position() so that both kinds of read are free of bank conflicts and P
// needs no exchange beyond movmatrix.
// Scales: the exponent of a key's row multiplies its scores; that of a value's row goes into the weight, P * 2^e. Weights are
// half precision, so what a row of queries puts its own against is the largest it has met of score + e, not of the score: its
// largest weight lies between 2^8 and 2^15, steps of half precision end at 2^-24, and what a weight may lose lies 2^33 below the
// row's own largest. What a row does not see, and value rows that have no weight in it, do not count. P itself, which is summed
// up in float, goes by the same reference (see below why float's range does). The rows of queries are scaled by powers of two to
// half precision, which holds all 8 bits of a bfloat16. Sums, maxima and accumulators are float.
#include <cooperative_groups.h>
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

// Positions of a tile: in clusters, and of the line, where a page (64) gives a warp twice the independent work at once.
constexpr int kClusterTile = 32;
__host__ __device__ constexpr int line_tile(int row_tiles) { return row_tiles == 1 ? 64 : 32; }
constexpr int kWarps = 8;                // of a CTA of a cluster
constexpr int kMaxCluster = 8;
constexpr int kWaitCode = 34;            // error word: a wait ran out
constexpr int kMaxSeqs = 4096;
constexpr int kMaxStages = 6;

// Warps of a CTA of the line, one CTA an SM: as many as registers allow (the state of a warp grows with its rows).
__host__ __device__ constexpr int line_warps(int row_tiles) { return row_tiles == 1 ? 12 : 8; }

// What the warp that begins a pair leaves for the join, by the pair's number.
struct Cut {
    int token0, kv_head, rows, first, last;     // first token (among the step's); rows of queries (0: the pair is not cut); warps
    int pad[3];
};

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
    int pairs;                           // what the host says there are
    int cluster, stages, tile_log;       // CTAs of a cluster (0: the line); tiles a warp keeps in flight; positions of a tile: 2^tile_log
    float scale_log2;
    Cut* cuts;                           // the line: [pairs]
    float* parts;                        // the line: [warps][2][rows][padded head size + 4]: values, then reference and sum
    int* error;
};

// The step's sequences in shared memory.
struct SeqTable {
    int *tiles_before, *pairs_before;    // [seqs + 1] tiles of the line, and pairs, before each
    int *start, *n, *slot;               // [seqs] position of the first new token, new tokens, slot
    __device__ __forceinline__ SeqTable(int* memory, int seqs)
        : tiles_before(memory), pairs_before(memory + seqs + 1), start(memory + 2 * (seqs + 1)), n(start + seqs), slot(n + seqs) {}
};
constexpr size_t seq_table_bytes(int seqs) { return ((size_t)5 * seqs + 2) * sizeof(int); }

// A sequence: every pair of it has as many tiles (a closed form keeps the line's arithmetic short): all from the first new token's
// window to the last new token, or, in a window, as many as a block's positions can touch, ending with the block's last one
// (but none before the sequence's first: of a block near it some lie behind the block and are masked away). Without a window
// the blocks of a long chunk are given its last tiles too, up to twice what they see; chunks that long go to the tcgen05 kernel
// where it takes their head size.
struct Seq {
    int start, n, blocks, first_tile, tiles;   // the sequence's first tile; tiles of one pair
    __device__ __forceinline__ int first_of(const AttnArgs& a, int token0) const {      // the first tile of the block of that token
        return max(first_tile, ((start + min(token0 + a.block_tokens, n) - 1) >> a.tile_log) - tiles + 1);
    }
};
__device__ __forceinline__ Seq seq_from(const AttnArgs& a, int start, int n) {
    Seq s;
    s.n = n;
    s.start = start;
    s.blocks = n <= 0 || n > a.most_new || start < 0 ? 0 : (n + a.block_tokens - 1) / a.block_tokens;
    s.first_tile = (a.window > 0 ? max(0, start - a.window + 1) : 0) >> a.tile_log;
    s.tiles = ((start + n - 1) >> a.tile_log) - s.first_tile + 1;
    if (a.window > 0 && a.window < start + n) s.tiles = min(s.tiles, ((a.window + a.block_tokens - 3) >> a.tile_log) + 2);
    return s;
}

// Fills the table (all threads of the CTA).
__device__ void scan_sequences(const AttnArgs& a, const SeqTable& table) {
    __shared__ int2 warp_total[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 carry = make_int2(0, 0);
    for (int base = 0; base < a.seqs; base += blockDim.x) {
        const int i = base + threadIdx.x;
        int2 mine = make_int2(0, 0);
        if (i < a.seqs) {
            const int n = a.cu[i + 1] - a.cu[i], start = a.seq_ends[i] - n;
            table.start[i] = start;
            table.n[i] = n;
            table.slot[i] = a.slot_ids[i];
            const Seq s = seq_from(a, start, n);
            mine.y = a.kv_heads * s.blocks;
            mine.x = mine.y * s.tiles;
        }
        int2 run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, run.x, o), y = __shfl_up_sync(0xffffffffu, run.y, o);
            if (lane >= o) { run.x += x; run.y += y; }
        }
        int2 before = carry;
        if (a.seqs > 32) {
            if (lane == 31) warp_total[warp] = run;
            __syncthreads();
            for (int w = 0; w < warps; ++w) {
                const int2 t = warp_total[w];
                if (w < warp) { before.x += t.x; before.y += t.y; }
                carry.x += t.x;
                carry.y += t.y;
            }
        }
        if (i < a.seqs) {
            table.tiles_before[i] = before.x + run.x - mine.x;
            table.pairs_before[i] = before.y + run.y - mine.y;
            if (i == a.seqs - 1) { table.tiles_before[a.seqs] = before.x + run.x; table.pairs_before[a.seqs] = before.y + run.y; }
        }
        __syncthreads();
    }
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
__device__ __forceinline__ int lds_u8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
    return (int)v;
}
__device__ __forceinline__ void sts_zero16(uint32_t addr) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Row r (0..15) of a block of 16 positions, as the tensor-core tile numbers them, is this position of the block: distinct
// modulo 8 among the rows that one ldmatrix phase reads, for the keys (rows 0-7, 8-15) and for the values (rows 0, 1, 8, 9,
// 2, 3, 10, 11, and the other eight).
__device__ __forceinline__ int row_position(int r) { return r < 8 ? r : 8 + ((r - 8) ^ 4); }

// With R a row's reference, the largest score + e so far rounded up, what is summed up is 2^(score - R + kSumShift), and the weight
// is that times 2^(e - kSumShift + 15 - kSlack). The reference moves where a score + e exceeds R + kSlack, so it seldom does, and
// weights are at most 2^15. e lies between -100 and 120 (kv_quant.cuh), and counts as at least kLeastCounted in R: so s, the largest
// score, has s - R between -121 and 86, and its 2^(s - R + kSumShift) lies between 2^-101, where a sum still has 2^-25 of it, and
// 2^106, of which a sum holds a million. Where all e are -100 the largest weight is at least 2^-12, a normal number of half precision.
constexpr int kSlack = 6, kSumShift = 20, kLeastCounted = -80;
constexpr float kUnit = 1 << (kSumShift - 15 + kSlack);          // what has been added up, over the sum, in these units is the output

// What a warp knows of the pair it works on, and what it has added up. NB: blocks of 64 of the head dimension; NHT: tiles
// of 8 rows of queries; BOX: head_dim is 64 * NB. A thread holds, of each tile of rows, rows 2 q4 and 2 q4 + 1 (q4 = lane % 4)
// and, of each 16 positions or dimensions, two (of positions: row_position(g) and row_position(g + 8), g = lane / 4).
template <int NB, int NHT, int FMT, bool BOX, int KT>
struct Rows {
    static constexpr int HDP = NB * 64, CH = HDP / 16, MT = KT / 16;       // padded head size, pieces of 16 dimensions
    uint32_t qf[CH][NHT][2];             // queries as half precision, scaled by a power of two to at most 2^11
    float q_scale[NHT][2];               // undoes the power of two, times scale * log2(e)
    float ot[CH][NHT][4];
    float limit[NHT][2], run_l[NHT][2];  // R + kSlack; the sum
    int first_pos, tokens, lowest;       // position of the first row's token, tokens, the lowest position that any sees
    uint32_t k_lane, v_lane;             // offsets in a tile of what this lane names in an ldmatrix of keys, of values

    // Row 0's place in q is `row0` (of rows of head_dim), row r's r / group tokens of `heads` rows and r % group further.
    __device__ __forceinline__ void begin(const AttnArgs& a, size_t row0, int first, int n_tokens) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
        const int hd = BOX ? HDP : a.head_dim, pieces = hd / 16, group = a.heads / a.kv_heads, rows = n_tokens * group;
        first_pos = first;
        tokens = n_tokens;
        lowest = a.window > 0 ? max(0, first - a.window + 1) : 0;
        // the row this lane names of 16 keys, and of a 16 x 16 block of values; lanes from 16 on name the next piece
        const int which = lane >> 4, at = lane & 15;
        const int k_row = row_position((lane & 7) + ((lane >> 3) & 1) * 8), v_row = row_position(2 * (at >> 2) + (at & 1) + ((at >> 1) & 1) * 8);
        k_lane = piece_at(hd, k_row, which);
        v_lane = (uint32_t)(KT * hd) + piece_at(hd, v_row, which);
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh) {
            const int r = nh * 8 + g;
            const __nv_bfloat16* src = a.q + (row0 + (size_t)(r / group) * a.heads + r % group) * hd;
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
                ot[c][nh][0] = ot[c][nh][1] = ot[c][nh][2] = ot[c][nh][3] = 0.f;
            }
            const float down = power_of_two(E - 10) * a.scale_log2;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                q_scale[nh][e] = __shfl_sync(0xffffffffu, down, (2 * q4 + e) * 4);
                limit[nh][e] = -CUDART_INF_F;
                run_l[nh][e] = 0.f;
            }
        }
    }

    // Shared-memory offset of a piece of 16 bytes of a row of a tile.
    static __device__ __forceinline__ uint32_t piece_at(int hd, int row, int piece) {
        if (BOX && NB == 2) return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
        if (BOX) return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
        return (uint32_t)(row * hd + (piece << 4));
    }

    // One tile: positions key0 .. key0 + KT - 1; shared-memory addresses of its codes (keys, then values) and exponents.
    __device__ __forceinline__ void tile(const AttnArgs& a, int key0, uint32_t codes, uint32_t exponents) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
        const int hd = BOX ? HDP : a.head_dim, pieces = hd / 16;
        const int last_pos = first_pos + tokens - 1;
        const uint32_t ks_lo = exponents + (uint32_t)g, ks_hi = exponents + (uint32_t)(8 + (g ^ 4));   // of the positions this thread holds
        const uint32_t ka = codes + k_lane, va = codes + v_lane;
        // The address for pieces c and c + 1 (c even) of the 16 rows from 16 mt on. In a box the pieces of a row are exchanged
        // by an exclusive or with bits of the row that 16 mt does not change.
        auto fragment_at = [&](uint32_t lane_at, int mt, int c) -> uint32_t {
            if (BOX) return (lane_at ^ (uint32_t)(c << 4)) + (uint32_t)(mt * 16 * HDP);
            const int which = lane >> 4;
            return lane_at + (uint32_t)(mt * 16 * hd) + (uint32_t)((min(c + which, pieces - 1) - which) << 4);     // (an odd last piece is read twice)
        };
        // every row sees every position of the tile, or a mask is needed
        const bool masked = key0 + KT - 1 > first_pos || (a.window > 0 && key0 <= last_pos - a.window);
        if (masked) {
            const int from = max(lowest - key0, 0), to = last_pos + 1 - key0;    // positions some row sees: [from, to)
            if (from > 0 || to < KT) {
                // value rows that no row sees may hold bytes that were never written: zeros (times zero weights)
                for (int idx = lane; idx < KT * pieces; idx += 32) {
                    const int row = idx / pieces, piece = idx - row * pieces;
                    if (row < from || row >= to) sts_zero16(codes + (uint32_t)(KT * hd) + piece_at(hd, row, piece));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
        }
        // S^T = K Q^T
        float st[MT][NHT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh) st[mt][nh][0] = st[mt][nh][1] = st[mt][nh][2] = st[mt][nh][3] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            if (!BOX && c >= pieces) break;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t w[4];       // rows 0-7 and 8-15 of piece c, then of piece c + 1
                ldmatrix_x4(w, fragment_at(ka, mt, c));
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
        // scores (in powers of two)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float f0 = scale_of(lds_u8(ks_lo + mt * 16)), f1 = scale_of(lds_u8(ks_hi + mt * 16));
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh) {
                st[mt][nh][0] *= f0 * q_scale[nh][0];
                st[mt][nh][1] *= f0 * q_scale[nh][1];
                st[mt][nh][2] *= f1 * q_scale[nh][0];
                st[mt][nh][3] *= f1 * q_scale[nh][1];
            }
        }
        if (masked) {
            const int group = a.heads / a.kv_heads;
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // the row sees the positions of the tile from `lo` to `hi`
                    const int hi = first_pos + min((nh * 8 + 2 * q4 + e) / group, tokens - 1) - key0, lo = a.window > 0 ? hi - a.window + 1 : 0;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const int x = mt * 16 + g, y = mt * 16 + 8 + (g ^ 4);
                        if (x > hi || x < lo) st[mt][nh][e] = -CUDART_INF_F;
                        if (y > hi || y < lo) st[mt][nh][e + 2] = -CUDART_INF_F;
                    }
                }
        }
        // whether any score + e exceeds its row's limit
        float e0[MT], e1[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            e0[mt] = (float)(max(lds_u8(ks_lo + KT + mt * 16) - 127, kLeastCounted));
            e1[mt] = (float)(max(lds_u8(ks_hi + KT + mt * 16) - 127, kLeastCounted));
        }
        bool moved = false;
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(st[0][nh][e] + e0[0], st[0][nh][e + 2] + e1[0]);
#pragma unroll
                for (int mt = 1; mt < MT; ++mt) x = fmax3(x, st[mt][nh][e] + e0[mt], st[mt][nh][e + 2] + e1[mt]);
                moved |= x > limit[nh][e];
            }
        if (__any_sync(0xffffffffu, moved)) {
            // a larger reference: what has been added up is put on the new footing (most tiles bring none, and then no maximum is
            // looked for among the threads)
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = st[0][nh][e] + e0[0];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) x = fmax3(x, st[mt][nh][e] + e0[mt], st[mt][nh][e + 2] + e1[mt]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = x > limit[nh][e] ? ceilf(x) + kSlack : limit[nh][e];
                    const float root = x == limit[nh][e] ? 1.f : ex2_approx(0.5f * (limit[nh][e] - x));
                    limit[nh][e] = x;
                    run_l[nh][e] = run_l[nh][e] * root * root;      // (a sum may have to go down by more than float has a factor for)
                    f[e] = root * root;
                }
#pragma unroll
                for (int c = 0; c < CH; ++c) { ot[c][nh][0] *= f[0]; ot[c][nh][1] *= f[1]; ot[c][nh][2] *= f[0]; ot[c][nh][3] *= f[1]; }
            }
        }
        // P, summed up, and the weights
        float ref[NHT][2];
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) ref[nh][e] = limit[nh][e] == -CUDART_INF_F ? 0.f : limit[nh][e] - (kSlack + kSumShift);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int b0 = lds_u8(ks_lo + KT + mt * 16), b1 = lds_u8(ks_hi + KT + mt * 16);
            const float w0 = b0 == kNoScale ? CUDART_NAN_F : __int_as_float(max(b0 - (kSumShift - 15 + kSlack), 0) << 23);
            const float w1 = b1 == kNoScale ? CUDART_NAN_F : __int_as_float(max(b1 - (kSumShift - 15 + kSlack), 0) << 23);
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = ex2_approx(st[mt][nh][e] - ref[nh][e & 1]);
                    run_l[nh][e & 1] += v;
                    // (a weight of zero stays zero whatever the byte of a position that is not seen says)
                    st[mt][nh][e] = masked && st[mt][nh][e] == -CUDART_INF_F ? 0.f : v * ((e & 2) ? w1 : w0);
                }
        }
        // ... as the B operand
        uint32_t pb[MT][NHT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nh = 0; nh < NHT; ++nh) {
                pb[mt][nh][0] = movmatrix_trans(pack_half2(st[mt][nh][0], st[mt][nh][1]));
                pb[mt][nh][1] = movmatrix_trans(pack_half2(st[mt][nh][2], st[mt][nh][3]));
            }
        // O^T += V^T P^T
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                if (!BOX && c >= pieces) break;
                uint32_t w[4];
                ldmatrix_bytes_trans_x2(w, fragment_at(va, mt, c));
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
    }

    // The end: sums over the threads that share a row.
    __device__ __forceinline__ void end() {
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = run_l[nh][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                run_l[nh][e] = l;
            }
    }
};

// A warp's tiles: places, copies and waits. A place is a row of the pools: pages of kv heads of 64 positions.
template <bool BOX, int KT>
struct Ring {
    const CUtensorMap *map_k, *map_v;
    uint64_t* bars;                      // [stages]
    uint32_t slots;                      // shared-memory address of [stages][keys | values]
    uint32_t scales;                     // ... of [stages][exponents of keys, of values]
    int stages, hd, tiles;               // tiles: the warp's
    int issued, used, stage;
    uint32_t parity;

    __device__ __forceinline__ uint32_t codes_at(int s) const { return slots + (uint32_t)(s * 2 * KT * hd); }
    __device__ __forceinline__ uint32_t scales_at(int s) const { return scales + (uint32_t)(s * 2 * KT); }
    __device__ __forceinline__ void request(const AttnArgs& a, int place, int into) {
        // (one lane for all four copies: those of several lanes would be issued one lane after the other)
        if ((threadIdx.x & 31) == 0) {
            const uint32_t bar = smem_u32(&bars[into]), dst = codes_at(into), sc = scales_at(into), bytes = (uint32_t)(KT * hd);
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * bytes + 2 * KT) : "memory");
            if (BOX) {
                asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                             ::"r"(dst), "l"(map_k), "r"(0), "r"(place), "r"(bar) : "memory");
                asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                             ::"r"(dst + bytes), "l"(map_v), "r"(0), "r"(place), "r"(bar) : "memory");
            } else {
                bulk(dst, a.k_codes + (size_t)place * hd, bytes, bar);
                bulk(dst + bytes, a.v_codes + (size_t)place * hd, bytes, bar);
            }
            bulk(sc, a.k_scale + place, KT, bar);
            bulk(sc + KT, a.v_scale + place, KT, bar);
        }
        ++issued;
    }
    static __device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
    }
    // Waits for the next tile (false: the limit ran out).
    __device__ __forceinline__ bool wait(const AttnArgs& a) {
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[stage], parity))) {
            if ((threadIdx.x & 31) == 0 && a.error) atomicExch(a.error, kWaitCode);
            return false;
        }
        ++used;
        return true;
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; parity ^= 1u; }
    }
    // What was asked for lands before the CTA gives up its shared memory.
    __device__ __forceinline__ void drain() {
        OutstandingFill left[8];
        const int n = outstanding_fills(issued, used, stages, left);
        for (int j = 0; j < n; ++j) mbar_wait(&bars[left[j].stage], left[j].parity);
    }
};
// The row of the pools of tile t (from the sequence's first) of sequence i and kv head kvh.
__device__ __forceinline__ int place_of(const AttnArgs& a, const SeqTable& table, int i, int tile, int kvh) {
    const int key = tile << a.tile_log;
    int page = a.pages.at(table.slot[i], key / kPageSize);
    if (page < 0) {
        if (a.error) atomicExch(a.error, kBadPlaceInAttention);
        page = 0;
    }
    return (page * a.kv_heads + kvh) * kPageSize + key % kPageSize;
}

__device__ __forceinline__ void store_row4(__nv_bfloat16* dst, float4 v, float by) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x * by, v.y * by), hi = __floats2bfloat162_rn(v.z * by, v.w * by);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
// How a part with reference (limit) m and sum l counts against the largest one, `top`: the root of the factor, to be applied twice,
// since a sum may have to go down by more than float has a factor for. (Without positions: 0; without a reference, because every
// score it saw is NaN: 1, and its sum is NaN.)
__device__ __forceinline__ float part_root(float m, float l, float top) {
    return m == -CUDART_INF_F ? (l == 0.f ? 0.f : 1.f) : ex2_approx(0.5f * (m - top));
}

// ---- clusters: blockIdx.x / cluster is the pair ---------------------------------------------------------------------------
template <int NB, int NHT, int FMT, bool BOX>
__global__ void __launch_bounds__(kWarps * 32) attention_quant_cluster_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                              const __grid_constant__ CUtensorMap map_v, AttnArgs a) {
    using R_ = Rows<NB, NHT, FMT, BOX, kClusterTile>;
    constexpr int HDP = R_::HDP, CH = R_::CH, LD = HDP + 4, R = 8 * NHT, kThreads = kWarps * 32;    // LD: a row of results (conflict-free)
    extern __shared__ __align__(16) unsigned char smem_raw[];
    namespace cg = cooperative_groups;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    const int hd = BOX ? HDP : a.head_dim, group = a.heads / a.kv_heads, S = a.stages, C = a.cluster;
    const size_t ring_bytes = (size_t)kWarps * S * 2 * kClusterTile * hd;
    unsigned char* ring0 = BOX ? reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) : smem_raw;
    float* wo = reinterpret_cast<float*>(ring0 + ring_bytes);       // [warp][R][LD] values
    float* wm = wo + kWarps * R * LD;                               // [warp][R] references, then the warps' factors
    float* wl = wm + kWarps * R;                                    // [warp][R] sums
    float* parts = wl + kWarps * R;                                 // the leader's: [C][R][LD] values, reference, sum
    float* end_of_parts = parts + (C > 1 ? C : 1) * R * LD;
    unsigned char* scales = reinterpret_cast<unsigned char*>(end_of_parts);
    uint64_t* bars = reinterpret_cast<uint64_t*>(scales + (size_t)kWarps * S * 2 * kClusterTile);
    const SeqTable table(reinterpret_cast<int*>(bars + kWarps * S), a.seqs);

    Ring<BOX, kClusterTile> ring{&map_k, &map_v, bars + warp * S, smem_u32(ring0 + (size_t)warp * S * 2 * kClusterTile * hd),
                                 smem_u32(scales + (size_t)warp * S * 2 * kClusterTile), S, hd, 0, 0, 0, 0, 0u};
    if (lane == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&ring.bars[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                  // q and the cache come from the kernels before
    pdl_launch_dependents();
    scan_sequences(a, table);
    const int pair_number = blockIdx.x / C, rank = blockIdx.x - pair_number * C;
    if (table.pairs_before[a.seqs] != a.pairs) {     // lengths on the device that are not those on the host: nothing is done
        if (threadIdx.x == 0 && a.error) atomicExch(a.error, kBadPlaceInAttention);
        return;                                      // (every CTA)
    }
    // (a CTA may write into the leader's memory only once the leader runs: arrived here, waited for below)
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int i = find_seq(table.pairs_before, a.seqs, pair_number);
    const Seq s = seq_from(a, table.start[i], table.n[i]);
    const int pair = pair_number - table.pairs_before[i], kvh = pair / s.blocks, token0 = (pair - kvh * s.blocks) * a.block_tokens;
    const int tokens = min(a.block_tokens, s.n - token0), rows = tokens * group;
    const size_t row0 = (size_t)(a.cu[i] + token0) * a.heads + (size_t)kvh * group;
    // this CTA's tiles, and of those the warp's: warp, warp + 8, ...
    const int per = (s.tiles + C - 1) / C, t_first = s.first_of(a, token0), t_lo = t_first + rank * per,
              t_hi = min(t_lo + per, t_first + s.tiles);
    ring.tiles = t_hi - t_lo > warp ? (t_hi - t_lo - warp + kWarps - 1) / kWarps : 0;
    // places are looked up 32 at once, a lane each
    auto look_up = [&](int first) { return first + lane < ring.tiles ? place_of(a, table, i, t_lo + warp + kWarps * (first + lane), kvh) : 0; };
    int places = look_up(0), looked = 0;
    auto request = [&](int k, int into) {
        if (k >= looked + 32) { looked += 32; places = look_up(looked); }
        ring.request(a, __shfl_sync(0xffffffffu, places, k - looked), into);
    };
    for (int k = 0; k < min(S, ring.tiles); ++k) request(k, k);

    R_ state;
    state.begin(a, row0, s.start + token0, tokens);
    bool ok = true;
    for (int k = 0; k < ring.tiles; ++k) {
        if (!(ok = ring.wait(a))) break;
        state.tile(a, (t_lo + warp + kWarps * k) * kClusterTile, ring.codes_at(ring.stage), ring.scales_at(ring.stage));
        __syncwarp();            // every lane has read the slot
        if (k + S < ring.tiles) request(k + S, ring.stage);
        ring.next();
    }
    if (!ok) ring.drain();

    // ---- the warps' results put together, then the CTAs' --------------------------------------------------------------
    {
        state.end();
        float* o = wo + (size_t)warp * R * LD;
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nh * 8 + 2 * q4 + e;
                if (g == 0) { wm[warp * R + r] = state.limit[nh][e]; wl[warp * R + r] = state.run_l[nh][e]; }
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    o[r * LD + c * 16 + g] = state.ot[c][nh][e];
                    o[r * LD + c * 16 + 8 + g] = state.ot[c][nh][2 + e];
                }
            }
    }
    const bool failed = __syncthreads_or(!ok) != 0;
    if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    float* mine = (C > 1 ? cluster.map_shared_rank(parts, 0) : parts) + (size_t)rank * R * LD;
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, wm[w * R + r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float root = part_root(wm[w * R + r], wl[w * R + r], m);
            l += wl[w * R + r] * root * root;
            wm[w * R + r] = root * root;
        }
        mine[r * LD + HDP] = m;
        mine[r * LD + HDP + 1] = failed ? CUDART_NAN_F : l;
    }
    __syncthreads();
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
        if (C > 1) *reinterpret_cast<float4*>(mine + (size_t)r * LD + d) = sum;
        else if (BOX || d < hd) store_row4(a.out + (row0 + (size_t)(r / group) * a.heads + r % group) * hd + d, sum, kUnit / parts[r * LD + HDP + 1]);
    }
    if (C == 1) return;
    cluster.sync();
    if (rank != 0) return;
    for (int idx = threadIdx.x; idx < rows * (HDP / 4); idx += kThreads) {
        const int r = idx / (HDP / 4), d = (idx - r * (HDP / 4)) * 4;
        float m = -CUDART_INF_F, l = 0.f;
        for (int c = 0; c < C; ++c) m = fmaxf(m, parts[((size_t)c * R + r) * LD + HDP]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < C; ++c) {
            const float* part = parts + ((size_t)c * R + r) * LD;
            const float root = part_root(part[HDP], part[HDP + 1], m), f = root * root;
            l += part[HDP + 1] * root * root;
            if (f == 0.f) continue;
            const float4 x = *reinterpret_cast<const float4*>(part + d);
            sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
        }
        if (BOX || d < hd) store_row4(a.out + (row0 + (size_t)(r / group) * a.heads + r % group) * hd + d, sum, kUnit / l);
    }
}

// ---- the line ---------------------------------------------------------------------------------------------------------------
template <int NB, int NHT, int FMT, bool BOX>
__global__ void __launch_bounds__(line_warps(NHT) * 32, 1) attention_quant_line_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                       const __grid_constant__ CUtensorMap map_v, AttnArgs a) {
    constexpr int KT = line_tile(NHT), W = line_warps(NHT);
    using R_ = Rows<NB, NHT, FMT, BOX, KT>;
    constexpr int HDP = R_::HDP, CH = R_::CH, LD = HDP + 4, R = 8 * NHT;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    const int hd = BOX ? HDP : a.head_dim, group = a.heads / a.kv_heads, S = a.stages;
    unsigned char* ring0 = BOX ? reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) : smem_raw;
    unsigned char* scales = ring0 + (size_t)W * S * 2 * KT * hd;
    uint64_t* bars = reinterpret_cast<uint64_t*>(scales + (size_t)W * S * 2 * KT);
    const SeqTable table(reinterpret_cast<int*>(bars + W * S), a.seqs);
    Ring<BOX, KT> ring{&map_k, &map_v, bars + warp * S, smem_u32(ring0 + (size_t)warp * S * 2 * KT * hd),
                       smem_u32(scales + (size_t)warp * S * 2 * KT), S, hd, 0, 0, 0, 0, 0u};
    if (lane == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&ring.bars[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                  // q and the cache come from the kernels before
    pdl_launch_dependents();
    scan_sequences(a, table);

    if (table.pairs_before[a.seqs] != a.pairs) {     // lengths on the device that are not those on the host: nothing is done
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0 && a.error) atomicExch(a.error, kBadPlaceInAttention);
            for (int i = threadIdx.x; i < a.pairs; i += W * 32) a.cuts[i].rows = 0;
        }
        return;                                      // (every CTA)
    }
    // this warp's run of the line (neighbouring runs on different SMs: the last ones may be empty)
    const int total = table.tiles_before[a.seqs], number = warp * gridDim.x + blockIdx.x, warps = W * gridDim.x;
    const int run = (total + warps - 1) / warps;
    const int u_lo = min(total, number * run), u_hi = min(total, u_lo + run);
    ring.tiles = u_hi - u_lo;
    auto look_up = [&](int first) -> int {
        if (first + lane >= ring.tiles) return 0;
        const int u = u_lo + first + lane, i = find_seq(table.tiles_before, a.seqs, u);
        const Seq s = seq_from(a, table.start[i], table.n[i]);
        const int pair = (u - table.tiles_before[i]) / s.tiles, t = u - table.tiles_before[i] - pair * s.tiles;
        const int kvh = pair / s.blocks;
        return place_of(a, table, i, s.first_of(a, (pair - kvh * s.blocks) * a.block_tokens) + t, kvh);
    };
    int places = look_up(0), looked = 0;
    auto request = [&](int k, int into) {
        if (k >= looked + 32) { looked += 32; places = look_up(looked); }
        ring.request(a, __shfl_sync(0xffffffffu, places, k - looked), into);
    };
    for (int k = 0; k < min(S, ring.tiles); ++k) request(k, k);

    bool ok = true;
    for (int u = u_lo; u < u_hi;) {
        // one part of one pair
        const int i = find_seq(table.tiles_before, a.seqs, u);
        const Seq s = seq_from(a, table.start[i], table.n[i]);
        const int pair = (u - table.tiles_before[i]) / s.tiles, kvh = pair / s.blocks, token0 = (pair - kvh * s.blocks) * a.block_tokens;
        const int pair_at = table.tiles_before[i] + pair * s.tiles, part_end = min(u_hi, pair_at + s.tiles);
        const int tokens = min(a.block_tokens, s.n - token0), rows = tokens * group;
        const int first_token = a.cu[i] + token0, first_tile = s.first_of(a, token0);
        const bool begins = pair_at >= u_lo, whole = begins && part_end == pair_at + s.tiles;
        // (a warp that gave up still says of the pairs it begins that there is nothing to join)
        if (begins && lane == 0)
            a.cuts[table.pairs_before[i] + pair] =
                Cut{first_token, kvh, whole || !ok ? 0 : rows, number, (pair_at + s.tiles - 1) / run, {0, 0, 0}};
        if (!ok) {
            u = part_end;
            continue;
        }
        R_ state;
        state.begin(a, (size_t)first_token * a.heads + (size_t)kvh * group, s.start + token0, tokens);
        for (; u < part_end; ++u) {
            if (!(ok = ring.wait(a))) break;
            state.tile(a, (first_tile + (u - pair_at)) * KT, ring.codes_at(ring.stage), ring.scales_at(ring.stage));
            __syncwarp();        // every lane has read the slot
            if (u - u_lo + S < ring.tiles) request(u - u_lo + S, ring.stage);
            ring.next();
        }
        if (!ok) {               // (the pair's rows are not valid: the error word says so)
            u = part_end;
            continue;
        }
        state.end();
        float* part = a.parts + ((size_t)number * 2 + (begins ? 1 : 0)) * R * LD;
#pragma unroll
        for (int nh = 0; nh < NHT; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nh * 8 + 2 * q4 + e;
                if (r >= rows) continue;
                if (whole) {
                    __nv_bfloat16* dst = a.out + ((size_t)(first_token + r / group) * a.heads + (size_t)kvh * group + r % group) * hd;
                    const float by = kUnit / state.run_l[nh][e];
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        if (BOX || c * 16 < hd) {
                            dst[c * 16 + g] = __float2bfloat16_rn(state.ot[c][nh][e] * by);
                            dst[c * 16 + 8 + g] = __float2bfloat16_rn(state.ot[c][nh][2 + e] * by);
                        }
                } else {
                    if (g == 0) { part[r * LD + HDP] = state.limit[nh][e]; part[r * LD + HDP + 1] = state.run_l[nh][e]; }
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        part[r * LD + c * 16 + g] = state.ot[c][nh][e];
                        part[r * LD + c * 16 + 8 + g] = state.ot[c][nh][2 + e];
                    }
                }
            }
    }
    if (!ok) ring.drain();
}

// Puts the parts of what was cut together, in the order of the line: P warps share a row of a pair (blockIdx.x), warp p of them
// takes its parts p, p + P, ..., lanes four dimensions each; then the P sums are added up. P follows the parts a pair is cut
// into, so that a warp's loads are under way together and warps have something to do (us a call, with P = 4 / 8 / 16: 7 parts,
// 64 sequences of 200 to 4,000 38.0 / 39.9 / 45.2; 14 parts 16.6 / 15.8 / 17.1; 28 parts 42.1 / 39.9 / 39.3; 55 parts, 8 x 32,000
// 59.8 / 56.8 / 54.3; 222 parts 75 / 62 / 50, with P = 32 48).
constexpr int join_warps(int P) { return P > 8 ? P : 8; }            // of a CTA
template <int HDP, int P>
__global__ void __launch_bounds__(join_warps(P) * 32) attention_quant_join_kernel(AttnArgs a, int rows_of_block) {
    constexpr int LD = HDP + 4, Q = HDP / 4, W = join_warps(P), kRowsOfCta = W / P;       // (16 or 32 lanes hold the dimensions)
    __shared__ float4 sums[W][Q];
    __shared__ float ms[W], ls[W];
    pdl_wait();              // (every CTA waits, those with nothing to do too: this kernel must not end before the one it follows)
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, p = warp % P;
    const int r = blockIdx.y * kRowsOfCta + warp / P, group = a.heads / a.kv_heads;
    const Cut cut = a.cuts[blockIdx.x];
    if (blockIdx.y * kRowsOfCta >= cut.rows) return;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < cut.rows) {
#pragma unroll 4
        for (int c = cut.first + p; c <= cut.last; c += P) {
            const float* part = a.parts + (((size_t)c * 2 + (c == cut.first ? 1 : 0)) * rows_of_block + r) * LD;
            const float pm = part[HDP], pl = part[HDP + 1];
            const float4 x = lane < Q ? *reinterpret_cast<const float4*>(part + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float top = fmaxf(m, pm);
            const float fr = part_root(m, l, top), hr = part_root(pm, pl, top), f = fr * fr, h = hr * hr;
            m = top;
            l = l * fr * fr + pl * hr * hr;
            o.x = o.x * f + x.x * h; o.y = o.y * f + x.y * h; o.z = o.z * f + x.z * h; o.w = o.w * f + x.w * h;
        }
    }
    if (lane < Q) sums[warp][lane] = o;
    if (lane == 0) { ms[warp] = m; ls[warp] = l; }
    __syncthreads();
    if (p != 0) return;
    m = ms[warp];
#pragma unroll
    for (int w = 1; w < P; ++w) m = fmaxf(m, ms[warp + w]);
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < P; ++w) {
        const float root = part_root(ms[warp + w], ls[warp + w], m), f = root * root;
        l += ls[warp + w] * root * root;
        if (f == 0.f || lane >= Q) continue;
        const float4 x = sums[warp + w][lane];
        o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
    }
    const int d = lane * 4;
    if (r < cut.rows && lane < Q && d < a.head_dim)
        store_row4(a.out + ((size_t)(cut.token0 + r / group) * a.heads + (size_t)cut.kv_head * group + r % group) * a.head_dim + d, o, kUnit / l);
}

constexpr int kDevices = 64;
int this_device() {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kDevices) throw std::runtime_error("attention_quant: more devices than it knows");
    return dev;
}
int sm_count() {
    static int known[kDevices] = {};
    const int dev = this_device();
    if (!known[dev]) cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev);
    return known[dev];
}
// Allows a kernel the shared memory it may ask for, once a device.
void allow_smem(const void* kernel, bool* prepared, size_t most) {
    const int dev = this_device();
    if (prepared[dev]) return;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) throw std::runtime_error(std::string("attention_quant: ") + cudaGetErrorString(e));
    prepared[dev] = true;
}

struct LaunchSizes {
    int pairs, rows_of_block, max_len;
};
constexpr size_t kRoom = 226 * 1024;     // shared memory of an SM, less what the system and the static part take

// Shared memory of a CTA: what it takes however many tiles are in flight (the step's sequences among it), and for one tile in
// flight a warp (codes, exponents, a barrier).
struct Smem {
    size_t fixed, a_tile;
    bool fits() const { return fixed + a_tile <= kRoom; }
};
Smem smem_of(int head_dim, int row_tiles, int seqs, int cluster) {
    const bool box = head_dim == 64 || head_dim == 128;
    const size_t R = 8 * row_tiles, LD = (head_dim <= 64 ? 64 : 128) + 4, warps = cluster ? kWarps : line_warps(row_tiles);
    const size_t tile = cluster ? kClusterTile : line_tile(row_tiles);
    return {(box ? 1024 : 0) + seq_table_bytes(seqs) + (cluster ? (kWarps * R * (LD + 2) + cluster * R * LD) * sizeof(float) : 0),
            warps * (2 * tile * (head_dim + 1) + sizeof(uint64_t))};
}

template <int NB, int NHT, int FMT, bool BOX>
void launch(AttnArgs a, const CUtensorMap& mk, const CUtensorMap& mv, const LaunchSizes& sizes, cudaStream_t stream) {
    constexpr int HDP = NB * 64, R = 8 * NHT;
    const Smem smem = smem_of(a.head_dim, NHT, a.seqs, a.cluster);
    if (!smem.fits())
        throw std::invalid_argument("attention_quant: " + std::to_string(a.seqs) + " sequences, head size " + std::to_string(a.head_dim) + ", " +
                                    std::to_string(NHT) + " tiles of rows and clusters of " + std::to_string(a.cluster) +
                                    " do not fit shared memory (attention_quant_fits)");
    const int room_for = (int)((kRoom - smem.fixed) / smem.a_tile);                    // tiles in flight
    if (a.cluster) {
        // as many tiles in flight as a warp gets, at most what is left
        const int tiles = ((sizes.max_len + kClusterTile - 1) / kClusterTile + 1 + a.cluster - 1) / a.cluster;
        a.stages = std::max(1, std::min({(tiles + kWarps - 1) / kWarps, kMaxStages, room_for}));
        static bool prepared[kDevices] = {};
        auto kernel = attention_quant_cluster_kernel<NB, NHT, FMT, BOX>;
        allow_smem((const void*)kernel, prepared, kRoom);
        note_launch();
        launch_kernel("attention_quant", kernel, dim3((unsigned)(sizes.pairs * a.cluster)), dim3(kWarps * 32), smem.fixed + a.stages * smem.a_tile,
                      stream, a.cluster, dependent_launch_enabled(), mk, mv, a);
        return;
    }
    constexpr int W = line_warps(NHT);
    a.stages = std::min(kMaxStages, room_for);
    static bool prepared[kDevices] = {};
    auto kernel = attention_quant_line_kernel<NB, NHT, FMT, BOX>;
    allow_smem((const void*)kernel, prepared, kRoom);
    note_launch(2);
    launch_kernel("attention_quant", kernel, dim3((unsigned)sm_count()), dim3(W * 32), smem.fixed + a.stages * smem.a_tile, stream, 1,
                  dependent_launch_enabled(), mk, mv, a);
    auto join = [&](auto kernel, int P) {
        const int rows_of_cta = join_warps(P) / P;
        launch_kernel("attention_quant", kernel, dim3((unsigned)sizes.pairs, (unsigned)((sizes.rows_of_block + rows_of_cta - 1) / rows_of_cta)),
                      dim3(join_warps(P) * 32), 0, stream, 1, dependent_launch_enabled(), a, R);
    };
    const int parts = sm_count() * W / sizes.pairs;          // of a pair
    if (parts <= 8) join(attention_quant_join_kernel<HDP, 4>, 4);
    else if (parts <= 20) join(attention_quant_join_kernel<HDP, 8>, 8);
    else if (parts <= 64) join(attention_quant_join_kernel<HDP, 16>, 16);
    else join(attention_quant_join_kernel<HDP, 32>, 32);
}

template <int FMT>
void launch_fmt(const AttnArgs& a, int row_tiles, const CUtensorMap& mk, const CUtensorMap& mv, const LaunchSizes& sizes, cudaStream_t stream) {
    const bool box = a.head_dim == 64 || a.head_dim == 128;
    auto pick = [&](auto small, auto boxed) { box ? boxed() : small(); };
#define SM_LAUNCH(NB, NHT) pick([&] { launch<NB, NHT, FMT, false>(a, mk, mv, sizes, stream); }, [&] { launch<NB, NHT, FMT, true>(a, mk, mv, sizes, stream); })
    if (a.head_dim <= 64) {
        if (row_tiles == 1) SM_LAUNCH(1, 1);
        else if (row_tiles == 2) SM_LAUNCH(1, 2);
        else SM_LAUNCH(1, 4);
    } else {
        if (row_tiles == 1) SM_LAUNCH(2, 1);
        else SM_LAUNCH(2, 2);
    }
#undef SM_LAUNCH
}

}  // namespace

bool attention_quant_supports(int heads, int kv_heads, int head_dim, long long pool_pages) {
    return head_dim % 16 == 0 && head_dim >= 16 && head_dim <= 128 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 &&
           pool_pages > 0 && pool_pages * kv_heads * kPageSize < (1ll << 31);
}

// Whether that many sequences' numbers fit beside the tiles.
bool attention_quant_fits(int head_dim, int row_tiles, int n_seqs, int cluster) {
    return n_seqs <= kMaxSeqs && smem_of(head_dim, row_tiles, n_seqs, cluster).fits();
}

// Floats of workspace that a launch needs: the line's cuts and parts.
long long attention_quant_workspace(int head_dim, int row_tiles, int pairs, int cluster) {
    if (cluster) return 0;
    const long long warps = (long long)sm_count() * line_warps(row_tiles);
    return warps * 2 * 8 * row_tiles * ((head_dim <= 64 ? 64 : 128) + 4) + (long long)pairs * (long long)(sizeof(Cut) / sizeof(float));
}

void attention_quant(const QuantPools& p, const void* q, void* out, int n_seqs, int heads, float scale, int window, const int32_t* slot_ids,
                     const int32_t* seq_ends, const int32_t* cu_seqlens, int max_len, int most_new, int row_tiles, int pairs, int cluster,
                     float* workspace, long long workspace_floats, int* error, cudaStream_t stream) {
    if (n_seqs <= 0 || pairs <= 0) return;
    const int kv_heads = p.kv_heads, head_dim = p.head_dim;
    if (!attention_quant_supports(heads, kv_heads, head_dim, p.pages))
        throw std::invalid_argument("attention_quant: " + std::to_string(heads) + " heads on " + std::to_string(kv_heads) + " of size " +
                                    std::to_string(head_dim) + " (multiples of 16 up to 128, at most 16 heads a kv head), or a pool of 2^31 rows");
    if (!(scale > 0.f) || !(scale < INFINITY)) throw std::invalid_argument("attention_quant: a scale of " + std::to_string(scale));
    if (cluster < 0 || cluster > kMaxCluster) throw std::invalid_argument("attention_quant: clusters of " + std::to_string(cluster) + " CTAs");
    if ((long long)pairs * std::max(cluster, 1) > 0x7fffffffll) throw std::invalid_argument("attention_quant: too many pairs for one launch");
    const int group = heads / kv_heads;
    if (n_seqs > kMaxSeqs) throw std::invalid_argument("attention_quant: more than " + std::to_string(kMaxSeqs) + " sequences");
    if ((row_tiles != 1 && row_tiles != 2 && (row_tiles != 4 || head_dim > 64)) || 8 * row_tiles < group)
        throw std::invalid_argument("attention_quant: " + std::to_string(row_tiles) + " tiles of rows");
    if (((uintptr_t)q | (uintptr_t)out) & 15 || ((uintptr_t)p.k_codes | (uintptr_t)p.v_codes | (uintptr_t)p.k_scale | (uintptr_t)p.v_scale) & 15)
        throw std::invalid_argument("attention_quant: operands must be 16-byte aligned");
    if (workspace_floats < attention_quant_workspace(head_dim, row_tiles, pairs, cluster)) throw std::invalid_argument("attention_quant: the workspace is too small");
    const int log_tile = (cluster ? kClusterTile : line_tile(row_tiles)) == 64 ? 6 : 5;
    AttnArgs a{(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)p.k_codes, (const uint8_t*)p.v_codes, (const uint8_t*)p.k_scale,
               (const uint8_t*)p.v_scale, {p.page_table, p.slots, p.table_stride, p.pages}, slot_ids, seq_ends, cu_seqlens, n_seqs, heads,
               kv_heads, head_dim, window, most_new, 8 * row_tiles / group, pairs, cluster, 0,
               log_tile, scale * 1.4426950408889634f, (Cut*)workspace,
               workspace + (cluster ? 0 : (long long)pairs * (long long)(sizeof(Cut) / sizeof(float))), error};
    CUtensorMap mk{}, mv{};
    if (head_dim == 64 || head_dim == 128) {
        // the pools as rows of codes; a box is a tile of positions of one kv head
        const CUtensorMapSwizzle swizzle = head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
        const uint64_t rows = (uint64_t)p.pages * kv_heads * kPageSize;
        mk = tiled_map_2d("attention_quant", CU_TENSOR_MAP_DATA_TYPE_UINT8, p.k_codes, (uint64_t)head_dim, rows, (uint64_t)head_dim, (uint32_t)head_dim,
                          1u << log_tile, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        mv = tiled_map_2d("attention_quant", CU_TENSOR_MAP_DATA_TYPE_UINT8, p.v_codes, (uint64_t)head_dim, rows, (uint64_t)head_dim, (uint32_t)head_dim,
                          1u << log_tile, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    const LaunchSizes sizes{pairs, a.block_tokens * group, max_len};
    if (p.fmt == QUANT_FP8) launch_fmt<QUANT_FP8>(a, row_tiles, mk, mv, sizes, stream);
    else if (p.fmt == QUANT_INT8) launch_fmt<QUANT_INT8>(a, row_tiles, mk, mv, sizes, stream);
    else throw std::invalid_argument("attention_quant: unknown format " + std::to_string(p.fmt));
}

}  // namespace sm
