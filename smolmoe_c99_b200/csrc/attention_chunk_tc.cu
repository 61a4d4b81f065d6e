// Causal attention of a chunk of new tokens per sequence over pages of bfloat16 keys and values (what an 8-bit cache stands
// for, read back page by page), head sizes 64 and 128, on the 5th-generation tensor cores.
//
// Rows of queries are (token, head of the group): the heads that share keys and values share a tile, so a tile of 128 rows is
// 128 / group tokens, keys are read once for all of them, and few rows lie beyond a tile's causal border. A CTA has two
// such tiles, A and B, under way: while the threads of one turn scores into weights, the tensor cores work for the other.
//   S_X = Q_X K^T    tcgen05.mma 128 x 128 x head_dim, both operands in shared memory, S (float) in tensor memory;
//   P_X = 2^(S * scale - reference) as bfloat16, back into tensor memory (a thread per row);
//   O_X += P_X V     tcgen05.mma 128 x head_dim x 128, P_X from tensor memory, V as it lies in memory (MN-major).
// Weights have the 8 bits of bfloat16, the sum takes them before they are rounded: at those sizes 0.0015 of the output away from 64
// bits, where the same in 32 bits, rounded once to bfloat16, is 0.0014 away.
// A row's reference is lazy: it moves when a tile's maximum exceeds it by more than 2^8, and only then is the accumulator
// rescaled.
//
// Tensor memory holds S (128 columns), P_A, P_B (64 each), O_A, O_B (128 each): the tiles take turns with one place for scores,
// free as soon as they are in the threads' registers, so S_B is computed while A's threads turn theirs into weights and the
// next S_A while B's do; the sums of values are issued by a warp of their own whenever weights are there. What was measured at
// 1,024 tokens of 28 heads of 128 onto 16,000 (249 GFLOP of products; us a call in one captured graph, reading the pages back and
// the join among them), in the order it was built: weights in the place of their
// scores, one thread issuing everything 278 us; the issuing warp's lanes together, one of them issuing 263; weights beside
// the scores 249; scores and sums issued by a warp each 241 (245 since the pages of several sequences lie packed). The products alone, with the same waits, take 177, and 223 with no
// exponentials: what is left is the way of a tile through its threads (read 64 KB of scores, largest, exponentials at 16 a cycle,
// write) and the turns with the one place. Two threads a row 247, a place for each tile's scores with heads of 64 115 against
// 107 (the tiles' threads then want the exponential unit at the same time), halves of 64 keys 414, part of the exponentials
// as polynomials and tiles issued by a warp each were slower too.
//
// Work is shared out as a line: the tiles of 128 keys of all pairs (two query tiles of one kv head), one after the other; each
// CTA of a grid of one an SM takes an equal run. What a run cuts is left as float accumulators, references and sums in a
// workspace and joined by a second kernel in the order of the line. So 512 tokens of 14 heads onto 8,000, 30 pairs, fill
// 148 SMs. Loads, products and row threads each go through the run at their own pace and meet at mbarriers only, so the next
// pair's queries and first scores come while the last weights of this one are under way. Lengths are read on the device: a
// captured launch follows a growing sequence.
//
// Every wait on an mbarrier is bounded; a wait that runs out records a code in *error and the CTA leaves without writing.
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

constexpr int kRows = 128, kKeys = 128;
constexpr int kRowWarps = 8;                // a thread a row: warps 0-3 tile A, 4-7 tile B
constexpr int kScoreWarp = 8, kSumWarp = 9, kLoadWarp = 10;     // Q K^T, P V, the copies
constexpr int kThreads = (kRowWarps + 3) * 32;
constexpr int kBlockBytes = 128 * 128;      // 128 rows of 128 bytes: one swizzled block of 64 bfloat16 columns
constexpr int kMaxSeqs = 1024, kMaxBlocks = 2048;

__host__ __device__ constexpr int stages_of(int head_dim) { return head_dim == 64 ? 4 : 2; }

// What the CTA that begins a pair leaves for the join, by the pair's number.
struct ChunkCut {
    int first_token, kv_head, tokens, first, last;     // tokens 0: the pair is not cut; CTAs
    int pad[3];
};

struct ChunkArgs {
    __nv_bfloat16* out;                  // [T, heads, HD]
    const int32_t* seq_ends;             // [seqs] lengths after the step
    const int32_t* cu;                   // [seqs + 1]
    int seqs, heads, kv_heads, window, skip_new, pages;    // pages: of the longest sequence, at most
    int room;                            // pages that were read back, at most
    int tile_tokens;                     // tokens of a tile of rows
    int blocks;                          // what the host says there are
    float scale_log2;
    ChunkCut* cuts;                      // [pairs]
    float* parts;                        // [CTAs][2][2 tiles][HD + 2][128 rows]
    int* error;
};

// The reduction dimension of V is its rows: an "MN-major" operand with 128-byte swizzle.
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)(kBlockBytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D += A B with A in tensor memory (two bfloat16 a column, a lane a row).
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32_raw(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
           "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
           "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// 16 float columns of this thread's lane back into tensor memory (complete after tmem_st_wait()).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
           "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A block: two tiles of rows of one sequence, for every kv head a pair of the line. Tiles of keys it sees: first .. first + n - 1.
struct Block {
    int token0, tokens, start;           // first token among the sequence's new ones, tokens (of both tiles), position of new token 0
    int first_tile, tiles;
};
__device__ __forceinline__ Block block_of(const ChunkArgs& a, int start, int n, int index) {
    Block b;
    b.start = start;
    b.token0 = index * 2 * a.tile_tokens;
    b.tokens = min(2 * a.tile_tokens, n - b.token0);
    const int lowest = a.window > 0 ? max(0, b.start + b.token0 - a.window + 1) : 0;
    b.first_tile = lowest / kKeys;
    b.tiles = (b.start + b.token0 + b.tokens - 1) / kKeys - b.first_tile + 1;
    return b;
}
// The last i with before[i] <= x.
__device__ __forceinline__ int find_last(const int* before, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}
// before[i] = the sum of values 0 .. i - 1 (value(i) is asked for by one thread), before[n] the total; all threads call it.
template <typename F>
__device__ void prefix_sums(int* before, int n, F value) {
    __shared__ int warp_total[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carry = 0;
    for (int base = 0; base < n; base += kThreads) {
        const int i = base + threadIdx.x, mine = i < n ? value(i) : 0;
        int run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += x;
        }
        if (lane == 31) warp_total[warp] = run;
        __syncthreads();
        int at = carry;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) at += warp_total[w];
            carry += warp_total[w];
        }
        if (i < n) before[i] = at + run - mine;
        __syncthreads();
    }
    if (threadIdx.x == 0) before[n] = carry;
    __syncthreads();
}

// The step's sequences and the line, in shared memory.
struct Line {
    int *blocks_before, *tiles_before;   // [seqs + 1] blocks before a sequence, [blocks + 1] tiles of the line before a block
    int *first, *start, *n;              // [seqs] first new token among the step's, its position, new tokens
    int* pages_before;                   // [seqs + 1] pages read back before those of a sequence
};
// One part of one pair: what a run holds of it.
struct Part {
    int kvh, number, pair_at, tiles;      // the pair's number, its place on the line, its tiles of keys
    int kt0, n_kt;                             // the part's tiles of keys
    int first_token, tokens, first_pos;
    int page0, last_page;                      // where page 0 of the sequence would lie; its last page
    int end;                                   // where the part ends on the line
};
__device__ __forceinline__ Part part_at(const ChunkArgs& a, const Line& line, int blocks, int u, int u_hi) {
    const int block_number = find_last(line.tiles_before, blocks, u), seq = find_last(line.blocks_before, a.seqs, block_number);
    const Block b = block_of(a, line.start[seq], line.n[seq], block_number - line.blocks_before[seq]);
    Part p;
    p.kvh = (u - line.tiles_before[block_number]) / b.tiles;
    p.number = block_number * a.kv_heads + p.kvh;
    p.pair_at = line.tiles_before[block_number] + p.kvh * b.tiles;
    p.tiles = b.tiles;
    p.end = min(u_hi, p.pair_at + b.tiles);
    p.n_kt = p.end - u;
    p.kt0 = b.first_tile + (u - p.pair_at);
    p.first_token = line.first[seq] + b.token0;
    p.tokens = b.tokens;
    p.first_pos = b.start + b.token0;
    p.page0 = line.pages_before[seq] - pages_read(b.start, b.start + line.n[seq], a.window, a.pages).first;
    p.last_page = (b.start + line.n[seq] - 1) / kPageSize;
    return p;
}

// A wait whose outcome is the warp's, so its lanes stay together where it runs out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attention_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v, ChunkArgs a, int least_run) {
    constexpr int DB = HD / 64, NS = stages_of(HD);
    constexpr int kTileBytes = DB * kBlockBytes;         // a tile of queries, of keys or of values
    constexpr uint32_t kTmemP = 128, kTmemO = 256;       // columns: S 0, P_A 128, P_B 192, O_A 256, O_B 384
    extern __shared__ uint8_t smem_raw[];
    uint8_t* q_s = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);   // [2 tiles][DB][128 rows][128 B]
    uint8_t* k_s = q_s + 2 * kTileBytes;                 // [NS][DB][128 keys][128 B]
    uint8_t* v_s = k_s + NS * kTileBytes;                // [NS]
    uint64_t* bars = (uint64_t*)(v_s + NS * kTileBytes);
    uint64_t *q_full = bars, *q_empty = bars + 1;        // a part's queries have landed; its last scores are done
    uint64_t* s_full = bars + 2;                         // [2 tiles] scores are in tensor memory
    uint64_t* p_full = bars + 4;                         // [2] weights are in tensor memory (and the accumulator is rescaled)
    uint64_t* pv_done = bars + 6;                        // [2] a PV is done: its weights' place is free, the accumulator whole
    uint64_t* o_empty = bars + 8;                        // [2] the part's accumulator has been read
    uint64_t* s_empty = bars + 10;                       // the scores have been read
    uint64_t* drain_bar = bars + 11;                     // [2] of each issuing warp
    uint64_t *k_full = bars + 13, *k_empty = k_full + NS, *v_full = k_empty + NS, *v_empty = v_full + NS;
    uint32_t* tmem_slot = (uint32_t*)(v_empty + NS);
    volatile int* failed = (volatile int*)(tmem_slot + 1);
    Line line;
    line.blocks_before = (int*)(tmem_slot + 2);
    line.first = line.blocks_before + a.seqs + 1;
    line.start = line.first + a.seqs;
    line.n = line.start + a.seqs;
    line.pages_before = line.n + a.seqs;
    line.tiles_before = line.pages_before + a.seqs + 1;

    const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads, tile_rows = a.tile_tokens * group;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);        // (a lane of each of the tile's warps)
            mbar_init(&pv_done[x], 1);
            mbar_init(&o_empty[x], 4);
        }
        mbar_init(s_empty, 4);
        mbar_init(&drain_bar[0], 1);
        mbar_init(&drain_bar[1], 1);
        for (int i = 0; i < 4 * NS; ++i) mbar_init(&k_full[i], 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kScoreWarp) tmem_alloc(tmem_slot, 512);
    // the rows of the query tiles that no copy fills: zeros
    for (int i = threadIdx.x; i < 2 * DB * (kRows - tile_rows) * 8; i += kThreads) {
        const int block = i / ((kRows - tile_rows) * 8), rest = i - block * (kRows - tile_rows) * 8;
        *reinterpret_cast<uint4*>(q_s + block * kBlockBytes + tile_rows * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();              // queries, pages and lengths come from the kernels before
    pdl_launch_dependents();

    prefix_sums(line.blocks_before, a.seqs, [&](int i) {
        const int first = a.cu[i], n = a.cu[i + 1] - first, end = a.seq_ends[i];
        line.first[i] = first;
        line.start[i] = end - n;
        line.n[i] = n;
        return n > a.skip_new && n <= end && end <= a.pages * kPageSize ? (n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens) : 0;
    });
    prefix_sums(line.pages_before, a.seqs, [&](int i) {
        return line.n[i] > a.skip_new ? pages_read(line.start[i], line.start[i] + line.n[i], a.window, a.pages).count : 0;
    });
    // (lengths on the device that are not those on the host, or pass the pages that were read back: nothing is done)
    const int blocks = line.blocks_before[a.seqs] == a.blocks && line.pages_before[a.seqs] <= a.room ? a.blocks : 0;
    if (blocks == 0 && blockIdx.x == 0) {
        if (threadIdx.x == 0 && a.error) atomicExch(a.error, kBadPlaceInAttention);
        for (int i = threadIdx.x; i < a.blocks * a.kv_heads; i += kThreads) a.cuts[i].tokens = 0;
    }
    prefix_sums(line.tiles_before, blocks, [&](int i) {
        const int seq = find_last(line.blocks_before, a.seqs, i);
        return a.kv_heads * block_of(a, line.start[seq], line.n[seq], i - line.blocks_before[seq]).tiles;
    });
    const int total = line.tiles_before[blocks], run = max((total + (int)gridDim.x - 1) / (int)gridDim.x, least_run);
    const int u_lo = min(total, (int)blockIdx.x * run), u_hi = min(total, u_lo + run);

    auto fail = [&](int code) {
        *failed = 1;
        if (a.error) atomicExch(a.error, code);
    };

    if (warp == kLoadWarp) {
        if ((threadIdx.x & 31) == 0) {
            bool ok = true;
            int f = 0, parts = 0, v_asked = 0;       // fills of K (as many of V, or one fewer), parts
            for (int u = u_lo; u < u_hi && ok;) {
                const Part p = part_at(a, line, blocks, u, u_hi);
                if (parts > 0 && !(ok = mbar_wait(q_empty, (uint32_t)(parts - 1) & 1u))) { fail(43); break; }
                const int both = p.tokens > a.tile_tokens ? 2 : 1;
                mbar_expect_tx(q_full, (uint32_t)(both * DB * tile_rows * 128));
                for (int x = 0; x < both; ++x)
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        tma_load_3d(q_s + x * kTileBytes + d * kBlockBytes, &map_q, d * 64, p.kvh * group, p.first_token + x * a.tile_tokens, q_full);
                ++parts;
                auto load = [&](uint8_t* dst, const CUtensorMap* map, int t, uint64_t* bar) {
                    mbar_expect_tx(bar, (uint32_t)kTileBytes);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // (a page the sequence does not hold is replaced by its last one: its rows are masked, but must be numbers)
                        const int row = ((p.page0 + min(2 * (p.kt0 + t) + half, p.last_page)) * a.kv_heads + p.kvh) * kPageSize;
#pragma unroll
                        for (int d = 0; d < DB; ++d) tma_load_2d(dst + d * kBlockBytes + half * (kBlockBytes / 2), map, d * 64, row, bar);
                    }
                };
                for (int t = 0; t < p.n_kt; ++t, ++f) {
                    const int s = f % NS;
                    if (f >= NS && !(ok = mbar_wait(&k_empty[s], (uint32_t)(f / NS - 1) & 1u))) { fail(41); break; }
                    load(k_s + s * kTileBytes, &map_k, t, &k_full[s]);
                    if (f >= NS && !(ok = mbar_wait(&v_empty[s], (uint32_t)(f / NS - 1) & 1u))) { fail(42); ++f; break; }
                    load(v_s + s * kTileBytes, &map_v, t, &v_full[s]);
                    ++v_asked;
                }
                u = p.end;
            }
            if (!ok || *failed) {
                // the way out: what was asked for lands before the CTA gives up its shared memory
                if (parts > 0) mbar_wait(q_full, (uint32_t)(parts - 1) & 1u);
                OutstandingFill left[8];
                int n = outstanding_fills(f, max(0, f - NS), NS, left);
                for (int i = 0; i < n; ++i) mbar_wait(&k_full[left[i].stage], left[i].parity);
                n = outstanding_fills(v_asked, max(0, v_asked - NS), NS, left);
                for (int i = 0; i < n; ++i) mbar_wait(&v_full[left[i].stage], left[i].parity);
            }
        }
    } else if (warp == kScoreWarp || warp == kSumWarp) {
        // A warp issues the scores' products, another the sums of values, each at its own pace. A warp's lanes go through the
        // run together and one of them issues: the operands of tcgen05.mma then stay in the warp's uniform registers. (With one
        // lane going through it all by itself a product took 80 cycles to issue against 64 to run.)
        auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
        const int lo = same(u_lo), hi = same(u_hi), role = same(warp - kScoreWarp);
        const uint32_t tm = (uint32_t)same((int)tmem);
        auto commit = [&](uint64_t* bar) {
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        struct Steps { int n_kt, both, end; };           // of a part: tiles of keys, tiles of rows, its end on the line
        auto steps_at = [&](int u) {
            const Part p = part_at(a, line, blocks, u, hi);
            return Steps{same(p.n_kt), same(p.tokens) > a.tile_tokens ? 2 : 1, same(p.end)};
        };
        bool ok = true;
        int f = 0;                                       // fills gone through
        if (role == 0) {
            const uint32_t idesc = instr_desc(kRows, kKeys);
            const uint64_t desc_q = smem_desc(smem_u32(q_s)), desc_k = smem_desc(smem_u32(k_s));
            int scored = 0, parts = 0;                   // times scores were computed, parts
            for (int u = lo; u < hi && ok; ++parts) {
                const Steps p = steps_at(u);
                u = p.end;
                if (!(ok = warp_wait(q_full, (uint32_t)parts & 1u))) { fail(51); break; }
                for (int t = 0; t < p.n_kt && ok; ++t, ++f) {
                    const int s = f % NS;
                    if (!(ok = warp_wait(&k_full[s], (uint32_t)(f / NS) & 1u))) { fail(45); break; }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (x >= p.both || !ok) continue;
                        // once the scores before these have been read
                        if (scored > 0 && !(ok = warp_wait(s_empty, (uint32_t)(scored - 1) & 1u))) { fail(52); continue; }
                        ++scored;
                        tc_fence_after();
                        const uint64_t q = desc_q + (uint64_t)(((uint32_t)x * kTileBytes) >> 4), k = desc_k + (uint64_t)(((uint32_t)s * kTileBytes) >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ++ks) {
                                const uint64_t off = (uint64_t)(((uint32_t)(ks / 4) * kBlockBytes + (uint32_t)(ks % 4) * 32) >> 4);
                                umma_bf16(tm, q + off, k + off, idesc, ks > 0 ? 1u : 0u);
                            }
                            umma_commit(&s_full[x]);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    commit(&k_empty[s]);
                    if (t + 1 == p.n_kt) commit(q_empty);
                }
            }
        } else {
            const uint32_t idesc = instr_desc(kRows, HD) | (1u << 16);     // V is MN-major
            const uint64_t desc_v = smem_desc_rows(smem_u32(v_s));
            int weights[2] = {0, 0}, ends[2] = {0, 0};   // tiles of keys and parts, of each tile of rows
            for (int u = lo; u < hi && ok;) {
                const Steps p = steps_at(u);
                u = p.end;
                for (int t = 0; t < p.n_kt && ok; ++t, ++f) {
                    const int s = f % NS;
                    if (!(ok = warp_wait(&v_full[s], (uint32_t)(f / NS) & 1u))) { fail(44); break; }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (x >= p.both || !ok) continue;
                        if (t == 0 && ends[x] > 0 && !(ok = warp_wait(&o_empty[x], (uint32_t)(ends[x] - 1) & 1u))) { fail(50); continue; }
                        if (!(ok = warp_wait(&p_full[x], (uint32_t)weights[x] & 1u))) { fail(46); continue; }
                        ++weights[x];
                        if (t + 1 == p.n_kt) ++ends[x];
                        tc_fence_after();
                        const uint64_t v = desc_v + (uint64_t)(((uint32_t)s * kTileBytes) >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < kKeys / 16; ++ks)
                                umma_bf16_ts(tm + kTmemO + (uint32_t)x * 128, tm + kTmemP + (uint32_t)x * 64 + (uint32_t)ks * 8,
                                             v + (uint64_t)(((uint32_t)ks * 16 * 128) >> 4), idesc, t == 0 && ks == 0 ? 0u : 1u);
                            umma_commit(&pv_done[x]);
                        }
                        __syncwarp();
                    }
                    if (ok) commit(&v_empty[s]);
                }
            }
        }
        if (__any_sync(0xffffffffu, !ok || *failed)) {   // no product is left under way
            commit(&drain_bar[role]);
            warp_wait(&drain_bar[role], 0);
        }
    } else {
        // ---- a thread a row ---------------------------------------------------------------------------------------------
        const int x = warp >> 2, quarter = warp & 3, row = quarter * 32 + (threadIdx.x & 31);
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t tmem_s = tmem + lane_base, tmem_p = tmem + kTmemP + (uint32_t)x * 64 + lane_base;       // scores; this tile's weights
        const uint32_t tmem_o = tmem + kTmemO + (uint32_t)x * 128 + lane_base;
        constexpr float kLazy = 8.0f;
        int tiles = 0;                       // of keys, of all parts
        bool ok = true;
        for (int u = u_lo; u < u_hi;) {
            const Part p = part_at(a, line, blocks, u, u_hi);
            // (a warp that gave up still says of the pairs that begin here that there is nothing to join)
            if (threadIdx.x == 0 && p.pair_at >= u_lo)
                a.cuts[p.number] = ChunkCut{p.first_token, p.kvh, p.end == p.pair_at + p.tiles || !ok ? 0 : p.tokens, (int)blockIdx.x, (p.pair_at + p.tiles - 1) / run, {0, 0, 0}};
            const bool whole = u == p.pair_at && p.end == p.pair_at + p.tiles;
            const int cut_slot = p.pair_at < u_lo ? 0 : 1;
            u = p.end;
            const int x_tokens = min(a.tile_tokens, p.tokens - x * a.tile_tokens);               // tokens of this tile of rows
            if (x_tokens <= 0 || !ok) continue;
            const int first_pos = p.first_pos + x * a.tile_tokens, last_pos = first_pos + x_tokens - 1;
            const int token = row / group, pos = first_pos + min(token, x_tokens - 1);
            float m = -CUDART_INF_F, l = 0.f;
            for (int t = 0; t < p.n_kt; ++t, ++tiles) {
                const int key0 = (p.kt0 + t) * kKeys;
                if (!warp_wait(&s_full[x], (uint32_t)tiles & 1u)) { fail(47); ok = false; break; }
                tc_fence_after();
                float sv[128];
                tmem_ld128(tmem_s, sv);
                tc_fence_before();
                warp_arrive(s_empty);
                // every row sees every key of the tile, or a mask is needed
                if (key0 + kKeys - 1 > first_pos || (a.window > 0 && key0 <= last_pos - a.window)) {
                    const int hi = pos - key0, lo = a.window > 0 ? hi - a.window + 1 : 0;        // this row's keys: lo .. hi
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (j > hi || j < lo) sv[j] = -CUDART_INF_F;
                }
                float top8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) top8[e] = fmaxf(sv[e], sv[8 + e]);
#pragma unroll
                for (int j = 16; j < 128; j += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top8[e] = fmax3(top8[e], sv[j + e], sv[j + 8 + e]);
                // maximum of the raw scores (the scale is positive)
                const float top = fmaxf(fmax3(top8[0], top8[1], top8[2]), fmax3(fmax3(top8[3], top8[4], top8[5]), top8[6], top8[7])) * a.scale_log2;
                // the PV before is done: the accumulator may be rescaled, and new weights written
                if (t > 0) {
                    if (!warp_wait(&pv_done[x], (uint32_t)(tiles - 1) & 1u)) { fail(49); ok = false; break; }
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, top > m + kLazy)) {
                    const float mx = fmaxf(m, top), corr = mx == -CUDART_INF_F ? 1.0f : ex2_approx(m - mx);
                    if (t > 0) {
#pragma unroll
                        for (int c = 0; c < HD / 16; ++c) {
                            float acc[16];
                            tmem_ld16(tmem_o + (uint32_t)(c * 16), acc);
#pragma unroll
                            for (int j = 0; j < 16; ++j) acc[j] *= corr;
                            tmem_st16(tmem_o + (uint32_t)(c * 16), acc);
                        }
                    }
                    l *= corr;
                    m = mx;
                }
                const float ref = m == -CUDART_INF_F ? 0.f : m;
                const uint64_t scale2 = pack_f32x2(a.scale_log2, a.scale_log2), ref2 = pack_f32x2(-ref, -ref);
                uint64_t sum2[2] = {0ull, 0ull};              // (the bits of two float zeros)
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t pk[32];
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        float x0, x1;
                        unpack_f32x2(fma_f32x2(pack_f32x2(sv[part * 64 + j], sv[part * 64 + j + 1]), scale2, ref2), x0, x1);
                        x0 = ex2_approx(x0);
                        x1 = ex2_approx(x1);
                        sum2[(j / 2) & 1] = add_f32x2(sum2[(j / 2) & 1], pack_f32x2(x0, x1));
                        pk[j / 2] = pack_bf16(x0, x1);
                    }
                    tmem_st32_raw(tmem_p + (uint32_t)(part * 32), pk);
                }
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(&p_full[x]);
                float lo2, hi2;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), lo2, hi2);
                l += lo2 + hi2;
            }
            if (ok && !warp_wait(&pv_done[x], (uint32_t)(tiles - 1) & 1u)) { fail(48); ok = false; }
            tc_fence_after();
            if (!__all_sync(0xffffffffu, ok && !*failed)) { ok = false; continue; }
            const bool live = token < x_tokens;
            const float inv = 1.0f / l;
            __nv_bfloat16* dst = a.out + ((size_t)(p.first_token + x * a.tile_tokens + token) * a.heads + (size_t)p.kvh * group + (row - token * group)) * HD;
            float* part = a.parts + (((size_t)blockIdx.x * 2 + cut_slot) * 2 + x) * (HD + 2) * kRows + row;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                float o[32];
                tmem_ld32(tmem_o + (uint32_t)(c * 32), o);
                if (c == HD / 32 - 1) {      // all of it has been read
                    tc_fence_before();
                    warp_arrive(&o_empty[x]);
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[(size_t)(c * 32 + i) * kRows] = o[i];
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4*>(dst + c * 32 + i) =
                            make_uint4(pack_bf16(o[i] * inv, o[i + 1] * inv), pack_bf16(o[i + 2] * inv, o[i + 3] * inv),
                                       pack_bf16(o[i + 4] * inv, o[i + 5] * inv), pack_bf16(o[i + 6] * inv, o[i + 7] * inv));
                }
            }
            if (!whole) {
                part[(size_t)HD * kRows] = m;
                part[(size_t)(HD + 1) * kRows] = l;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kScoreWarp) tmem_dealloc(tmem, 512);
}

// How a part with maximum m and sum l counts against the maximum `top` of all. (No key seen: 0; no maximum, because every
// score is NaN: 1, and the sum is NaN.)
__device__ __forceinline__ float part_factor(float m, float l, float top) { return m == -CUDART_INF_F ? (l == 0.f ? 0.f : 1.f) : ex2_approx(m - top); }

// Puts the parts of a cut pair together, in the order of the line: blockIdx.x a tile of rows of a pair, blockIdx.y eight of its
// dimensions, P threads a row, which take every P-th part, four under way together; their sums are then added up. P follows the
// parts a pair is cut into (us a call with P = 1 / 2 / 4 / 8: about 5 parts, six windowed sequences 41.9 / 44.2 / 49.5 / 59.7; 13 parts,
// 200 tokens onto 1,000 21.2 / 19.9 / 18.5 / 21.1; 19 parts, 128 onto 8,000 30.2 / 25.9 / 24.9 / 26.6).
constexpr int kJoinDims = 8, kJoinParts = 4;
template <int HD, int P>
__global__ void __launch_bounds__(P * kRows) attention_chunk_join_kernel(ChunkArgs a) {
    __shared__ float sums[P > 1 ? P : 1][P > 1 ? kJoinDims + 2 : 1][kRows];
    pdl_wait();              // (every CTA waits: this kernel must not end before the one it follows)
    pdl_launch_dependents();
    const ChunkCut cut = a.cuts[blockIdx.x >> 1];
    const int group = a.heads / a.kv_heads, x = blockIdx.x & 1, row = threadIdx.x % kRows, p = threadIdx.x / kRows, token = row / group;
    const int tokens = min(a.tile_tokens, cut.tokens - x * a.tile_tokens);
    if (tokens <= 0) return;
    const bool live = token < tokens;
    const float* first = a.parts + (size_t)x * (HD + 2) * kRows + row;
    const size_t stride = (size_t)2 * (HD + 2) * kRows;                 // of a part of both tiles; two a CTA
    float m = -CUDART_INF_F, l = 0.f, o[kJoinDims];
#pragma unroll
    for (int i = 0; i < kJoinDims; ++i) o[i] = 0.f;
    auto add = [&](float pm, float pl, const float (&v)[kJoinDims]) {
        const float top = fmaxf(m, pm), f = part_factor(m, l, top), g = part_factor(pm, pl, top);
        m = top;
        l = l * f + pl * g;
#pragma unroll
        for (int i = 0; i < kJoinDims; ++i) o[i] = o[i] * f + v[i] * g;
    };
    if (live)
        for (int c0 = cut.first + p; c0 <= cut.last; c0 += P * kJoinParts) {
            float pm[kJoinParts], pl[kJoinParts], v[kJoinParts][kJoinDims];
#pragma unroll
            for (int k = 0; k < kJoinParts; ++k) {
                const int c = min(c0 + k * P, cut.last);
                const float* part = first + ((size_t)c * 2 + (c == cut.first ? 1 : 0)) * stride;
                pm[k] = part[(size_t)HD * kRows];
                pl[k] = part[(size_t)(HD + 1) * kRows];
#pragma unroll
                for (int i = 0; i < kJoinDims; ++i) v[k][i] = part[(size_t)(blockIdx.y * kJoinDims + i) * kRows];
            }
#pragma unroll
            for (int k = 0; k < kJoinParts; ++k)
                if (c0 + k * P <= cut.last) add(pm[k], pl[k], v[k]);
        }
    if (P > 1) {
        if (p > 0) {
            sums[p][kJoinDims][row] = m;
            sums[p][kJoinDims + 1][row] = l;
#pragma unroll
            for (int i = 0; i < kJoinDims; ++i) sums[p][i][row] = o[i];
        }
        __syncthreads();
        if (p > 0) return;
#pragma unroll
        for (int q = 1; q < P; ++q) {
            float v[kJoinDims];
#pragma unroll
            for (int i = 0; i < kJoinDims; ++i) v[i] = sums[q][i][row];
            add(sums[q][kJoinDims][row], sums[q][kJoinDims + 1][row], v);
        }
    }
    if (!live) return;
    const float inv = 1.0f / l;
    __nv_bfloat16* dst = a.out + ((size_t)(cut.first_token + x * a.tile_tokens + token) * a.heads + (size_t)cut.kv_head * group + (row - token * group)) * HD +
                         blockIdx.y * kJoinDims;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv), pack_bf16(o[4] * inv, o[5] * inv),
                                                pack_bf16(o[6] * inv, o[7] * inv));
}

constexpr int kDevices = 64;
int this_device() {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kDevices) throw std::runtime_error("attention_chunk: more devices than it knows");
    return dev;
}
int sm_count() {
    static int known[kDevices] = {};
    const int dev = this_device();
    if (!known[dev]) cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev);
    return known[dev];
}

template <int HD>
void launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkArgs& a, int blocks, int least_run, cudaStream_t stream) {
    constexpr int NS = stages_of(HD);
    const size_t smem = 1024 + (size_t)(2 + 2 * NS) * (HD / 64) * kBlockBytes + (13 + 4 * NS) * sizeof(uint64_t) + 8 +
                        (size_t)(5 * a.seqs + blocks + 3) * sizeof(int);
    auto kernel = attention_chunk_kernel<HD>;
    static bool prepared[kDevices] = {};
    const int dev = this_device();
    if (!prepared[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
        if (e != cudaSuccess) throw std::runtime_error(std::string("attention_chunk: ") + cudaGetErrorString(e));
        prepared[dev] = true;
    }
    note_launch(2);
    launch_kernel("attention_chunk", kernel, dim3((unsigned)sm_count()), dim3(kThreads), smem, stream, 1, dependent_launch_enabled(), mq, mk, mv, a, least_run);
    auto join = [&](auto kernel, int P) {
        launch_kernel("attention_chunk", kernel, dim3((unsigned)(blocks * a.kv_heads * 2), HD / kJoinDims), dim3(P * kRows), 0, stream, 1, dependent_launch_enabled(), a);
    };
    const int parts = sm_count() / (blocks * a.kv_heads) + 1;     // of a pair, about
    if (parts <= 6) join(attention_chunk_join_kernel<HD, 1>, 1);
    else if (parts <= 9) join(attention_chunk_join_kernel<HD, 2>, 2);
    else join(attention_chunk_join_kernel<HD, 4>, 4);
}

}  // namespace

bool attention_chunk_supports(int heads, int kv_heads, int head_dim, long long pool_pages, int n_seqs, int blocks) {
    return (head_dim == 64 || head_dim == 128) && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 && pool_pages > 0 &&
           pool_pages * kv_heads * kPageSize < (1ll << 31) && n_seqs <= kMaxSeqs && blocks <= kMaxBlocks;
}

long long attention_chunk_workspace(int head_dim, int kv_heads, int blocks) {
    return (long long)blocks * kv_heads * (long long)(sizeof(ChunkCut) / sizeof(float)) + (long long)sm_count() * 2 * 2 * (head_dim + 2) * kRows;
}

void attention_chunk(const void* q, void* out, int T, int n_seqs, int heads, int kv_heads, int head_dim, float scale, int window, const void* k_pages,
                     const void* v_pages, int pages, long long room, const int32_t* seq_ends, const int32_t* cu_seqlens, int skip_new, int blocks, float* workspace,
                     long long workspace_floats, int* error, cudaStream_t stream) {
    if (n_seqs <= 0 || blocks <= 0 || T <= 0) return;
    if (!attention_chunk_supports(heads, kv_heads, head_dim, room, n_seqs, blocks))
        throw std::invalid_argument("attention_chunk: " + std::to_string(heads) + " heads on " + std::to_string(kv_heads) + " of size " +
                                    std::to_string(head_dim) + " (64 or 128, at most 16 heads a kv head), " + std::to_string(n_seqs) + " sequences, " +
                                    std::to_string(blocks) + " blocks of queries");
    if (!(scale > 0.f) || !(scale < INFINITY)) throw std::invalid_argument("attention_chunk: a scale of " + std::to_string(scale));
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15)
        throw std::invalid_argument("attention_chunk: operands must be 16-byte aligned");
    if (workspace_floats < attention_chunk_workspace(head_dim, kv_heads, blocks)) throw std::invalid_argument("attention_chunk: the workspace is too small");
    const int group = heads / kv_heads, tile_tokens = kRows / group;
    // queries as [T][heads][head_dim]: a box is 64 columns of a group's heads of a tile's tokens
    CUtensorMap mq;
    cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)heads * head_dim * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tile_tokens}, step[3] = {1, 1, 1};
    const CUresult r = tensor_map_encoder()(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("attention_chunk: cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
    // pages [room, kv heads, 64 positions, head_dim] as rows of head_dim: a box is 64 columns of a page of one kv head
    const uint64_t rows = (uint64_t)room * kv_heads * kPageSize;
    const CUtensorMap mk = tiled_map_2d("attention_chunk", CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, k_pages, (uint64_t)head_dim, rows, (uint64_t)head_dim * 2, 64,
                                        kPageSize, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    const CUtensorMap mv = tiled_map_2d("attention_chunk", CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v_pages, (uint64_t)head_dim, rows, (uint64_t)head_dim * 2, 64,
                                        kPageSize, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    ChunkCut* cuts = (ChunkCut*)workspace;
    ChunkArgs a{(__nv_bfloat16*)out, seq_ends, cu_seqlens, n_seqs, heads, kv_heads, window, skip_new, pages, (int)room, tile_tokens, blocks, scale * 1.4426950408889634f, cuts,
                workspace + (long long)blocks * kv_heads * (long long)(sizeof(ChunkCut) / sizeof(float)), error};
    // a run is at least this many tiles: a part costs about as much as one to leave and join
    const int least_run = 2;
    if (head_dim == 64) launch<64>(mq, mk, mv, a, blocks, least_run, stream);
    else launch<128>(mq, mk, mv, a, blocks, least_run, stream);
}

}  // namespace sm
