// Grouped product of two MXFP4 operands on the block-scaled tensor cores.
//
//   out^T[n, t] = sum_b 2^(ws[n,b] + xs[t,b] - 254) sum_{i<32} w[n, 32b+i] * x[t, 32b+i]
//
// (accumulator lane = weight row n, column = token t.)  Nothing is decoded: the packed e2m1 bytes of both operands go
// from global memory into shared memory by TMA and from there into tcgen05.mma.kind::mxf4.block_scale, which multiplies
// 64 contraction elements per instruction, applies both e8m0 exponents per 32 elements and accumulates in fp32.  A
// zero element times any finite scale is zero, so ragged ends need no mask: TMA fills what lies outside the tensors
// with zero bytes.  An exponent byte of 255 is NaN, as the OCP format has it.
//
// Roles (512 threads, one CTA per SM, persistent):
//   warp 0      TMA producer: per stage of 256 contraction elements (128 bytes a row, 128-byte swizzle) the weight tile
//               [rows_w x 128 B] and the item's activation rows in boxes of xbox rows
//   warp 1      MMA issuer: tcgen05.cp of the stage's scales shared memory -> tensor memory (32 lanes
//               x 16 bytes, replicated to the four lane quarters), then up to four MMAs of 64 elements
//   warps 2-7   scales, a span of 1024 elements (32 exponent bytes a row, four stages) at a time in a ring of two: every
//               thread has two of the 128 + 256 rows and reads a row's 32 bytes with two 16-byte loads (three where rows
//               do not start on 16 bytes: gpt-oss has 90 bytes a row, which is also why they cannot come by TMA), those
//               of the next span in flight, and the next item's on their way to L2, while a span is written as the 4-byte words of 128 elements that tcgen05.cp
//               takes (row r at (r % 32) * 16 + (r / 32) * 4; a warp's 32 rows are eight of each quarter, so that no two
//               lanes share a bank).  What counts here is the number of instructions: a warp issues one every five or six
//               cycles, and all of a span's have to fit the 2000 cycles that the tensor cores take for it
//   warps 8-15  epilogue, two per TMEM lane quarter taking alternate 32-token chunks, as in tensor_fwd_kernel.cuh
//
// CG = 2 (long groups): a cluster of two CTAs shares every item -- same rows, neighbouring weight tiles, 256 x 256
// multiplied by one tcgen05.mma.cta_group::2 that the leader issues.  Each CTA loads its own weight tile and half of the
// activation rows, 32 KiB a stage instead of 48 for the same product: what bounds long groups is L2 -> shared memory
// (about 47 bytes per cycle and SM).  Each keeps the scales of its weight rows and of all activation rows; the leader's
// tcgen05.cp.cta_group::2 copies both CTAs' into their own tensor memory.  The peer's MMA warp forwards "my tiles have
// landed" to the leader; completions are committed to both.
//
// Work item = (group, balanced chunk of <= tok_cap rows, rows_w weight rows), weight tile fastest.  With few rows per
// group the kernel streams weights and rows_w < 128 evens out the items over the SMs (the MMA still multiplies 128
// lanes; the lanes above rows_w hold stale bytes and scales and are not read back).
//
// Measured (kernel alone, graphs of 20 launches): gpt-oss gate_up (N = 5760, K = 2880, 32 experts) 4 rows each 55 us, 5.1 TB/s;
// 1024 rows each 281-308 us, 3.9-3.5 PFLOP/s; Qwen3 gate_up (N = 1536, K = 2048, 128 experts) 256 rows each 70-79 us, 2.9-2.6
// PFLOP/s (the lower figures at 1.65 GHz, where the power limit then holds the clock); one gpt-oss token through 4 experts
// 13 us.  (The W4A16 kernels here: 252, 1115, 218 us for the first three, 12 for the last.)
// What bounds it: with few rows the issuer, 635 cycles per stage at about 31 per tcgen05 instruction and 130 per completed
// barrier (without the MMAs and copies 47 us of the 55, the rate of a plain copy); with 256 rows the tiles' way from L2 into
// shared memory, 45 to 49 bytes per cycle and SM (without MMAs and copies 58 us of 70; in pairs, measured on 8 x 2048 rows,
// K = 7168, which the rule gives to single CTAs, 170 of 203), and the power limit; scales take 3 to 9 % (rows on 16 bytes the
// less).  A launch reaches its first MMA after 3.5 us with few rows (1.6 of them launch and group table) and after 6 with
// many, when every SM loads at once.
#pragma once

#include "tensor_fwd_kernel.cuh"

namespace gnf4b {

constexpr int kQStageK = 256;                  // contraction elements per stage
constexpr int kQRowBytes = kQStageK / 2;       // 128 bytes: one swizzle row
constexpr int kQWTile = 128 * kQRowBytes;      // 16 KiB, whatever rows_w: the MMA reads 128 rows
constexpr int kQMaxStages = 12;
constexpr int kQMaxGroups = 256;               // groups per launch (longer lists take several)
constexpr int kQScaleWarps = 6, kQEpiWarps = 8;      // 16 warps in all: 128 registers a thread
constexpr int kQEpiChunks = 4;                 // 32-token chunks per epilogue warp, at most
constexpr int kQScaleWarp0 = 2, kQEpiWarp0 = kQScaleWarp0 + kQScaleWarps;
constexpr int kQThreads = (kQEpiWarp0 + kQEpiWarps) * 32;
constexpr int kQTmemCols = 512;
constexpr int kQTableBytes = kQMaxGroups * 16 + (kQMaxGroups + 1) * 4 + 16 * 4 + 4;

struct W4A4Args {
    const uint8_t* xs;          // activation scales, rows of K / 32 bytes
    const uint8_t* ws;          // weight scales, byte strides ws_se, ws_sn
    const int32_t* off;
    const int32_t* eids;
    int32_t* status;
    uint16_t* out;
    int64_t ws_se, ws_sn;
    int64_t T, N, K;
    int32_t G, E;
    int32_t rows_w;             // weight rows per item, a multiple of 8, <= 128
    FastDiv n_tiles;            // items per chunk: ceil(N / rows_w), in a pair ceil(N / 256)
    int32_t k_stages;           // ceil(K / 256)
    int32_t tok_cap;            // activation rows per item, a multiple of 16 (in a pair 32), <= 256
    int32_t xbox;               // activation rows per TMA box
    int32_t x_bytes;            // shared memory of a stage's activations, whole boxes
    int32_t stages;
    int32_t acc_bufs;           // 1 or 2 accumulators
    int32_t x_blocks;           // ceil(tok_cap / 128): 512-byte scale blocks per 128 elements
};

// scales of 128 elements: [weights 512 B][activations x_blocks * 512 B]; eight of these are a span
__host__ __device__ inline int w4a4_half_bytes(int x_blocks) { return 512 * (1 + x_blocks); }
__host__ __device__ inline int w4a4_span_bytes(int x_blocks) { return 8 * w4a4_half_bytes(x_blocks); }
__host__ __device__ inline size_t w4a4_fixed_bytes(int x_blocks) {
    return 1024 /*alignment*/ + 2 * (size_t)w4a4_span_bytes(x_blocks) + kQTableBytes + 512 /*barriers*/;
}

__device__ __forceinline__ void tma_load_3d(void* dst_smem, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst_smem)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tc_mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                            uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows x 16 bytes of shared memory -> 4 tensor-memory columns, the same 32 lanes in each of the four lane quarters
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t s_desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(s_desc) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// descriptor of that source: no swizzle, 8-row groups of 128 bytes one after the other
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3fffu) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// kind::mxf4 instruction descriptor: e2m1 x e2m1, both K-major, e8m0 scales, M = m; the byte pair of the 4-byte
// scale words that belongs to this instruction's 64 elements is 0 or 2
__device__ __forceinline__ uint32_t mxf4_idesc(uint32_t m, uint32_t n_umma, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n_umma >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (sf_id << 29);
}

// ---- the same over a CTA pair
__device__ __forceinline__ void tc_mma_mxf4_2(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_cp_scales_2(uint32_t taddr, uint64_t s_desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(s_desc) : "memory");
}
__device__ __forceinline__ void tmem_alloc_2(uint32_t* dst_smem, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_2(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// arrive on a barrier of the cluster and publish what this thread wrote (the scales)
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
template <int CG>
__device__ __forceinline__ void q_mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (CG == 2) tc_mma_mxf4_2(d, ad, bd, idesc, sfa, sfb, accumulate);
    else tc_mma_mxf4(d, ad, bd, idesc, sfa, sfb, accumulate);
}
template <int CG>
__device__ __forceinline__ void q_cp(uint32_t taddr, uint64_t s_desc) {
    if (CG == 2) tc_cp_scales_2(taddr, s_desc);
    else tc_cp_scales(taddr, s_desc);
}
// commit to this CTA's barrier, in a pair to the peer's too (peer_off: its shared::cluster address minus this one's)
template <int CG>
__device__ __forceinline__ void q_commit(uint64_t* bar, uint32_t peer_base, uint32_t own_base) {
    if (CG == 2) {
        tc_commit2(smem_u32(bar));
        tc_commit2(peer_base + (smem_u32(bar) - own_base));
    } else {
        tc_commit(bar);
    }
}
template <int CG>
__device__ __forceinline__ bool q_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return CG == 2 ? mbar_wait_bounded_cluster(bar, parity, abort_flag) : mbar_wait_bounded(bar, parity, abort_flag);
}

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// one lane of the warp, always the same one
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct QGroup {
    int32_t row0, rows, eid, chunk_rows;
};
struct QTable {
    const QGroup* grp;       // [G]
    const uint32_t* base;    // [G + 1] items before group g (the host sees to it that all items fit 31 bits)
};
struct QItem {
    int32_t row0, tokens, eid, n0;
};

// Item `id` -> its group, chunk and tile; g: the group of an earlier item.  Called by whole warps.
__device__ __forceinline__ bool next_qitem(const W4A4Args& a, const QTable& tb, int32_t& g, uint32_t id, QItem* it, int32_t tile_rows,
                                           int32_t tile_first) {
    // all lanes together, 32 groups at a time: one after the other, the dozen groups between two items of an SM cost
    // every role two thousand cycles per item
    while (true) {
        const int32_t next = g + 1 + (int32_t)(threadIdx.x & 31);
        const uint32_t past = __ballot_sync(0xffffffffu, next <= a.G && id >= tb.base[next]);      // a run from lane 0 on
        g += __popc(past);
        if (past != 0xffffffffu) break;
    }
    if (g >= a.G) return false;
    const QGroup gr = tb.grp[g];
    const uint32_t local = id - tb.base[g];
    const uint32_t mc = a.n_tiles.div(local);       // n0: of the item; a pair's second CTA adds 128
    it->row0 = gr.row0 + (int32_t)mc * gr.chunk_rows;
    it->tokens = min(gr.chunk_rows, gr.row0 + gr.rows - it->row0);
    it->eid = gr.eid;
    it->n0 = (int32_t)(local - mc * a.n_tiles.d) * tile_rows + tile_first;
    return true;
}

// Thread t takes groups 2t and 2t + 1: item counts, then a block-wide inclusive scan.  Groups with a bad expert id or
// bad offsets are flagged in the status word and get no items.
__device__ __forceinline__ void build_qtable(const W4A4Args& a, QGroup* grp, uint32_t* base, uint32_t* warp_tot) {
    static_assert(kQThreads * 2 >= kQMaxGroups, "one thread per two groups");
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    uint32_t items[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int g = 2 * t + h;
        if (g >= a.G) continue;
        QGroup gr;
        gr.row0 = __ldg(a.off + g);
        const int64_t rows = (int64_t)__ldg(a.off + g + 1) - gr.row0;
        gr.eid = __ldg(a.eids + g);
        const bool pad = gr.eid == GNF4B_PAD_EXPERT;     // padding group: skipped, not an error
        const bool bad_e = (gr.eid < 0 || gr.eid >= a.E) && !pad;
        const bool bad_o = rows < 0 || gr.row0 < 0 || gr.row0 + rows > a.T;
        if ((bad_e || bad_o) && rows != 0 && a.status && blockIdx.x == 0)
            atomicOr(a.status, bad_e ? GNF4B_ST_BAD_EXPERT : GNF4B_ST_BAD_OFFSETS);
        gr.rows = (pad || bad_e || bad_o) ? 0 : (int32_t)rows;
        // equal chunks, a multiple of 16 rows each (a 64-bit division here costs every launch a third of a microsecond)
        const uint32_t r = (uint32_t)gr.rows;
        if (r <= (uint32_t)a.tok_cap) {
            gr.chunk_rows = r ? (int32_t)((r + 15u) & ~15u) : 16;
            items[h] = r ? a.n_tiles.d : 0u;
        } else {
            const uint32_t chunks = (r + (uint32_t)a.tok_cap - 1u) / (uint32_t)a.tok_cap;
            const uint32_t each = ((r + chunks - 1u) / chunks + 15u) & ~15u;
            gr.chunk_rows = (int32_t)each;
            items[h] = (r + each - 1u) / each * a.n_tiles.d;
        }
        grp[g] = gr;
    }
    // saturating at 2^31 - 1: offsets that go back and forth can name the same rows in many groups, more items than the
    // host has counted, and a wrapped number would be taken for an item of another group
    const auto add = [](uint32_t x, uint32_t y) { return min(x + y, 0x7fffffffu); };
    uint32_t incl = add(items[0], items[1]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl = add(incl, up);
    }
    if (lane == 31) warp_tot[w] = incl;
    uint32_t excl = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) excl = 0;
    __syncthreads();
    for (int v = 0; v < w; ++v) excl = add(excl, warp_tot[v]);
    if (2 * t < a.G) base[2 * t + 1] = add(excl, items[0]);
    if (2 * t + 1 < a.G) base[2 * t + 2] = add(add(excl, items[0]), items[1]);
    if (t == 0) base[0] = 0;
}

// The aligned 16 bytes at q as far as they lie in the scale tensor [lo, hi), zeros elsewhere: for the pieces of its first
// and last rows.
__device__ __noinline__ uint4 load_scale_edge(const uint8_t* q, const uint8_t* lo, const uint8_t* hi) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 16; ++b)
        if (q + b >= lo && q + b < hi) w[b >> 2] |= (uint32_t)__ldg(q + b) << (8 * (b & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The 32 bytes at offset `at` (0..15) of the 48 in raw as 8 words, zeros behind the first `valid`.
__device__ __forceinline__ void align_scale_row(const uint32_t* raw, uint32_t at, int valid, uint32_t* out) {
    uint32_t w[9];
    const bool by2 = at & 8, by1 = at & 4;
#pragma unroll
    for (int j = 0; j < 9; ++j) {
        const uint32_t v0 = by2 ? raw[j + 2] : raw[j];
        const uint32_t v1 = j + 3 < 12 ? (by2 ? raw[j + 3] : raw[j + 1]) : 0u;
        w[j] = by1 ? v1 : v0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = __funnelshift_r(w[j], w[j + 1], 8 * (at & 3));
    if (valid < 32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int left = valid - 4 * j;
            out[j] = left >= 4 ? out[j] : left <= 0 ? 0u : out[j] & ((1u << (8 * left)) - 1u);
        }
    }
}

template <int CG>
__global__ void __launch_bounds__(kQThreads, 1)
w4a4_kernel(const __grid_constant__ W4A4Args a, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    // tiles of all stages (each a multiple of 1024 bytes), then two spans of scales, then the tables
    const int tile_bytes = kQWTile + a.x_bytes;
    const int half_bytes = w4a4_half_bytes(a.x_blocks), span_bytes = 8 * half_bytes;
    uint8_t* s_scale = smem + (size_t)a.stages * tile_bytes;
    uint8_t* grp_raw = s_scale + 2 * (size_t)span_bytes;
    QGroup* s_grp = reinterpret_cast<QGroup*>(grp_raw);
    uint32_t* s_base = reinterpret_cast<uint32_t*>(grp_raw + kQMaxGroups * 16);
    uint32_t* s_wtot = s_base + kQMaxGroups + 1;
    // full[s]: tiles landed (TMA bytes + the producer's arrival); done[s]: the stage's copies and MMAs have completed,
    // its shared memory and its tensor-memory scale slot may be refilled; sc_full / sc_done: the same for a span of scales
    uint64_t* full = reinterpret_cast<uint64_t*>(grp_raw + ((kQTableBytes + 15) & ~15));
    uint64_t* done = full + kQMaxStages;
    uint64_t* acc_full = done + kQMaxStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* sc_full = acc_empty + 2;
    uint64_t* sc_done = sc_full + 2;
    uint64_t* landed = sc_done + 2;                        // the peer's own tiles, forwarded to the leader's full[]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(landed + kQMaxStages);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = uniform(threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const uint32_t stages = (uint32_t)a.stages;
    const uint32_t rank = CG == 2 ? (uint32_t)uniform((int)cluster_ctarank()) : 0u;
    const uint32_t worker = CG == 2 ? blockIdx.x >> 1 : blockIdx.x, workers = CG == 2 ? gridDim.x >> 1 : gridDim.x;
    const int32_t tile_rows = CG == 2 ? 256 : a.rows_w, tile_first = (int32_t)rank * 128;
    if (threadIdx.x == 32) {         // the descriptors are launch parameters: on their way before anything else
        tma_prefetch_map(&x_map);
        tma_prefetch_map(&w_map);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kQMaxStages; ++s) {
            mbar_init(full + s, CG);
            mbar_init(done + s, 1);
            mbar_init(landed + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + b, 1);
            mbar_init(acc_empty + b, kQEpiWarps * CG);
            mbar_init(sc_full + b, kQScaleWarps + (CG == 2 && rank == 0 ? 1 : 0));
            mbar_init(sc_done + b, 1);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        if (CG == 2) {
            tmem_alloc_2(tmem_slot, kQTmemCols);
        } else {
            tmem_alloc(tmem_slot, kQTmemCols);
            tmem_relinquish();
        }
    }
    pdl_wait();                      // group tables, operands and the output belong to earlier kernels until here
    pdl_launch_dependents();         // not before: a successor may read, ahead of its own wait, what OUR predecessor wrote
    build_qtable(a, s_grp, s_base, s_wtot);
    const QTable tb{s_grp, s_base};
    tc_fence_before();
    if (CG == 2) cluster_sync_all();      // the peer's barriers exist before anything arrives on them
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t own_base = smem_u32(full);
    const uint32_t leader_base = CG == 2 ? map_to_cta(own_base, 0) : 0u, peer_base = CG == 2 ? map_to_cta(own_base, 1) : 0u;
    const uint32_t tmem_sf0 = tmem_base + (uint32_t)(a.acc_bufs * a.tok_cap);      // scale slots behind the accumulators
    const uint32_t slot_cols = 8u * (1u + (uint32_t)a.x_blocks);

    // The producer's and the issuer's loops are run by their whole warp, every loop condition a vote, with one elected
    // lane around the instructions: TMA and tcgen05 instructions take their operands from uniform registers, and in
    // control flow that the compiler cannot see to be the same for all lanes every one of them is preceded by a chain of
    // moves into those -- about 100 cycles per instruction, which alone made a stage take 1 us whatever its size.
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        int32_t g = 0;
        QItem it;
        uint32_t s = 0, phase = 0, id = worker;
        while (__all_sync(0xffffffffu, next_qitem(a, tb, g, id, &it, tile_rows, tile_first))) {
            // a pair's CTA loads half of the MMA's rows (32 and its multiples, so that a half is a multiple of 16)
            const int half = CG == 2 ? ((uniform(it.tokens) + 31) & ~31) >> 1 : 0;
            const int row0 = uniform(it.row0) + (CG == 2 ? (int)rank * half : 0), n0 = uniform(it.n0), eid = uniform(it.eid);
            const int boxes = ((CG == 2 ? half : uniform(it.tokens)) + a.xbox - 1) / a.xbox;
            uint64_t* const bars = CG == 2 && rank == 1 ? landed : full;
            const uint32_t bytes = (uint32_t)((a.rows_w + boxes * a.xbox) * kQRowBytes);
            bool ok = true;
            for (int rb = 0; rb < a.k_stages; ++rb) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(done + s, phase ^ 1, abort_flag));   // the first round passes at once
                if (!ok) break;
                if (elect_one()) {
                    uint8_t* st = smem + (size_t)s * tile_bytes;
                    mbar_arrive_expect_tx(bars + s, bytes);
                    tma_load_3d(st, &w_map, rb * kQRowBytes, n0, eid, bars + s);
                    for (int b = 0; b < boxes; ++b)
                        tma_load_2d(st + kQWTile + b * a.xbox * kQRowBytes, &x_map, rb * kQRowBytes, row0 + b * a.xbox, bars + s);
                }
                if (++s == stages) { s = 0; phase ^= 1; }
            }
            if (!ok) break;
            id += workers;
        }
    } else if (warp == 1 && rank == 1) {
        // ------------------------------------------------------------ the pair's second CTA: tiles landed and scales
        // written -> leader.  The scale warps' stores are published to the tensor core that reads them, this SM's own, by
        // their proxy fence; a release at cluster scope in every one of them would cost a thousand cycles per span
        int32_t g = 0;
        QItem it;
        uint32_t s = 0, phase = 0, sp = 0, sp_phase = 0, id = worker;
        while (__all_sync(0xffffffffu, next_qitem(a, tb, g, id, &it, tile_rows, tile_first))) {
            bool ok = true;
            for (int rb = 0; rb < a.k_stages; ++rb) {
                if ((rb & 3) == 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(sc_full + sp, sp_phase, abort_flag));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_release_cluster(leader_base + (smem_u32(sc_full + sp) - own_base));
                    sp ^= 1;
                    sp_phase ^= sp ^ 1;
                }
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(landed + s, phase, abort_flag));
                if (!ok) break;
                if (lane == 0) mbar_arrive_cluster(leader_base + s * 8);
                if (++s == stages) { s = 0; phase ^= 1; }
            }
            if (!ok) break;
            id += workers;
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        int32_t g = 0;
        QItem it;
        uint32_t s = 0, phase = 0, buf = 0, acc_phase = 0, sp = 0, sp_phase = 0, id = worker;
        const uint32_t half_cols = 4u * (1u + (uint32_t)a.x_blocks);
        const uint64_t w_desc0 = umma_desc(smem_u32(smem), 16, 1024), sc_desc0 = scale_desc(smem_u32(s_scale));
        const uint32_t tile_step = (uint32_t)tile_bytes >> 4, half_step = (uint32_t)half_bytes >> 4, span_step = (uint32_t)span_bytes >> 4;
        const int tail = (int)((a.K - (int64_t)(a.k_stages - 1) * kQStageK + 63) >> 6);   // 64-element steps of the last stage
        while (__all_sync(0xffffffffu, next_qitem(a, tb, g, id, &it, tile_rows, tile_first))) {
            const uint32_t tokens = (uint32_t)uniform(it.tokens);
            const uint32_t n_umma = CG == 2 ? (tokens + 31u) & ~31u : (tokens + 15u) & ~15u;
            const uint32_t id0 = mxf4_idesc(128 * CG, n_umma, 0), id2 = mxf4_idesc(128 * CG, n_umma, 2);
            const bool two = tokens > 128u;
            const uint32_t acc = tmem_base + buf * (uint32_t)a.tok_cap;
            bool ok = __all_sync(0xffffffffu, q_wait<CG>(acc_empty + buf, acc_phase ^ 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            for (int rb0 = 0; ok && rb0 < a.k_stages; rb0 += 4) {
                ok = __all_sync(0xffffffffu, q_wait<CG>(sc_full + sp, sp_phase, abort_flag));
                const uint64_t src0 = sc_desc0 + sp * span_step;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int rb = rb0 + i;
                    if (rb >= a.k_stages) break;
                    ok = __all_sync(0xffffffffu, ok && q_wait<CG>(full + s, phase, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    const bool last = rb + 1 == a.k_stages;
                    const int steps = last ? tail : 4;      // steps that exist (a trailing half step is zero elements)
                    const uint64_t da = w_desc0 + s * tile_step, db = da + (kQWTile >> 4), src = src0 + 2 * i * half_step;
                    const uint32_t sf = tmem_sf0 + s * slot_cols, sf1 = sf + half_cols;
                    if (elect_one()) {
                        q_cp<CG>(sf, src);
                        q_cp<CG>(sf + 4, src + (512 >> 4));
                        if (two) q_cp<CG>(sf + 8, src + (1024 >> 4));
                        q_mma<CG>(acc, da, db, id0, sf, sf + 4, rb > 0 ? 1u : 0u);
                        if (steps > 1) q_mma<CG>(acc, da + 2, db + 2, id2, sf, sf + 4, 1u);
                        if (steps > 2) {
                            q_cp<CG>(sf1, src + half_step);
                            q_cp<CG>(sf1 + 4, src + half_step + (512 >> 4));
                            if (two) q_cp<CG>(sf1 + 8, src + half_step + (1024 >> 4));
                            q_mma<CG>(acc, da + 4, db + 4, id0, sf1, sf1 + 4, 1u);
                            if (steps > 3) q_mma<CG>(acc, da + 6, db + 6, id2, sf1, sf1 + 4, 1u);
                        }
                        q_commit<CG>(done + s, peer_base, own_base);
                        if (i == 3 || last) q_commit<CG>(sc_done + sp, peer_base, own_base);
                        if (last) q_commit<CG>(acc_full + buf, peer_base, own_base);
                    }
                    if (++s == stages) { s = 0; phase ^= 1; }
                }
                sp ^= 1;
                sp_phase ^= sp ^ 1;
            }
            if (!ok) break;
            if (++buf == (uint32_t)a.acc_bufs) { buf = 0; acc_phase ^= 1; }
            id += workers;
        }
    } else if (warp < kQEpiWarp0) {
        // ------------------------------------------------------------ scales: global -> registers -> shared memory
        // Blocks of 32 rows: 0..3 the weight tile's, 4..11 the activations'; block b of its 128 rows is rows 8b .. 8b + 7 of
        // each quarter.  This warp has blocks sw and sw + 6.
        const int sw = warp - kQScaleWarp0;
        const int quarter = lane >> 3;
        const int64_t kb = a.K / 32;
        const uint8_t* w_hi = a.ws + (int64_t)(a.E - 1) * a.ws_se + (a.N - 1) * a.ws_sn + kb;
        const uint8_t* x_hi = a.xs + a.T * kb;
        const uintptr_t places = reinterpret_cast<uintptr_t>(a.ws) | reinterpret_cast<uintptr_t>(a.xs) | (uintptr_t)kb | (uintptr_t)a.ws_sn |
                                 (uintptr_t)a.ws_se;
        const bool aligned = (places & 15) == 0, aligned8 = (places & 7) == 0;       // every row starts on 16 / on 8 bytes
        const int spans = (a.k_stages + 3) >> 2;
        int32_t g = 0;
        QItem it;
        uint32_t id = worker;
        bool have = __all_sync(0xffffffffu, next_qitem(a, tb, g, id, &it, tile_rows, tile_first));
        int sp = 0;
        const uint8_t* row[2] = {nullptr, nullptr};         // this lane's rows; those that do not exist read the last that does
        uint32_t at[2] = {0, 0};                            // their place in 16 bytes
        uint32_t here = 0;                                  // one bit per block: it has rows
        int inside[2] = {0, 0};                             // spans whose 48 bytes all lie in the tensor
        uint32_t raw[2][12], raw_at[2] = {0, 0};            // a span's bytes as loaded, and where they begin
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int j = 0; j < 12; ++j) raw[o][j] = 0;
        // a new item: its rows, and their first bytes on the way to L2 a whole span before they are loaded
        auto enter = [&]() {
            if (!have) return;
            here = 0;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const int b = sw + o * kQScaleWarps;
                const bool w = b < 4;
                const int first = 8 * (b & 3);
                const int rows = w ? (int)min((int64_t)a.rows_w, a.N - it.n0) : it.tokens - ((b >> 2) - 1) * 128;
                if (first >= rows) continue;
                here |= 1u << o;
                const int r = min(quarter * 32 + first + (lane & 7), rows - 1);
                const uint8_t* base = w ? a.ws + (int64_t)it.eid * a.ws_se + (int64_t)it.n0 * a.ws_sn
                                        : a.xs + ((int64_t)it.row0 + ((b >> 2) - 1) * 128) * kb;
                const int64_t pitch = w ? a.ws_sn : kb;
                row[o] = base + r * pitch;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(row[o]));
                at[o] = (uint32_t)(reinterpret_cast<uintptr_t>(row[o]) & 15);
                const uint8_t* last = base + min(127, rows - 1) * pitch;
                inside[o] = base - (reinterpret_cast<uintptr_t>(base) & 15) >= (w ? a.ws : a.xs)
                                ? (int)min((int64_t)spans, ((w ? w_hi : x_hi) - last - 16) >> 5) : 0;
            }
        };
        enter();
        // the next span of this CTA's items; returns its bytes per row (0: none) and which blocks it has
        auto fetch = [&](uint32_t& blocks) -> int {
            if (!have) return 0;
            const int valid = (int)min((int64_t)32, kb - (int64_t)sp * 32);
            blocks = here;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                if (!(here >> o & 1u)) continue;
                const uint8_t* p = row[o] + sp * 32;
                raw_at[o] = at[o];
                if (aligned) {
                    const uint4 v0 = __ldg(reinterpret_cast<const uint4*>(p));
                    const uint4 v1 = __ldg(reinterpret_cast<const uint4*>(p) + (valid > 16 ? 1 : 0));
                    raw[o][0] = v0.x; raw[o][1] = v0.y; raw[o][2] = v0.z; raw[o][3] = v0.w;
                    raw[o][4] = v1.x; raw[o][5] = v1.y; raw[o][6] = v1.z; raw[o][7] = v1.w;
                } else {
                    const uint4* q = reinterpret_cast<const uint4*>(p - at[o]);
                    uint4 v0, v1, v2;
                    if (sp < inside[o]) {
                        v0 = __ldg(q); v1 = __ldg(q + 1);
                        v2 = make_uint4(0, 0, 0, 0);          // (not v1, which would have to arrive first)
                        if (valid + (aligned8 ? 8 : 15) > 32) v2 = __ldg(q + 2);
                    } else {
                        const bool w = sw + o * kQScaleWarps < 4;
                        const uint8_t* lo = w ? a.ws : a.xs;
                        const uint8_t* hi = w ? w_hi : x_hi;
                        v0 = load_scale_edge(reinterpret_cast<const uint8_t*>(q), lo, hi);
                        v1 = load_scale_edge(reinterpret_cast<const uint8_t*>(q + 1), lo, hi);
                        v2 = load_scale_edge(reinterpret_cast<const uint8_t*>(q + 2), lo, hi);
                    }
                    raw[o][0] = v0.x; raw[o][1] = v0.y; raw[o][2] = v0.z; raw[o][3] = v0.w;
                    raw[o][4] = v1.x; raw[o][5] = v1.y; raw[o][6] = v1.z; raw[o][7] = v1.w;
                    raw[o][8] = v2.x; raw[o][9] = v2.y; raw[o][10] = v2.z; raw[o][11] = v2.w;
                }
            }
            if (++sp == spans) {
                sp = 0;
                id += workers;
                have = __all_sync(0xffffffffu, next_qitem(a, tb, g, id, &it, tile_rows, tile_first));
                enter();
            }
            return valid;
        };
        uint32_t slot = 0, phase = 0, blocks = 0;
        int valid = fetch(blocks);
        while (valid) {
            // rows behind the last hold bytes of other rows: they belong to accumulator entries that nobody reads
            uint32_t out[2][8];
            const uint32_t put = blocks;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                if (!(put >> o & 1u)) continue;
                if (aligned && valid >= 32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[o][j] = raw[o][j];
                } else if (aligned8) {                      // 280 cycles instead of 540 a span with few rows
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[o][j] = 4 * j < valid ? ((raw_at[o] & 8) ? raw[o][j + 2] : raw[o][j]) : 0u;
                } else {
                    align_scale_row(raw[o], raw_at[o], valid, out[o]);
                }
            }
            valid = fetch(blocks);                          // on its way while this span waits for its slot and is written
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(sc_done + slot, phase ^ 1, abort_flag))) break;
            uint8_t* dst0 = s_scale + slot * span_bytes + (lane & 7) * 16 + quarter * 4;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                if (!(put >> o & 1u)) continue;
                const int b = sw + o * kQScaleWarps;
                uint8_t* dst = dst0 + (b >> 2) * 512 + (b & 3) * 128;
#pragma unroll
                for (int j = 0; j < 8; ++j) *reinterpret_cast<uint32_t*>(dst + j * half_bytes) = out[o][j];
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(sc_full + slot);     // in a pair the second CTA's MMA warp passes it on
            slot ^= 1;
            phase ^= slot ^ 1;
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3;
        const int e = (warp - kQEpiWarp0) >> 2;              // takes chunks e, e + 2, ...
        int32_t g = 0;
        QItem it;
        uint32_t buf = 0, acc_phase = 0;
        bool ok = true;
        const bool pair_ok = (a.N % 2) == 0;
        for (uint32_t id = worker; ok && next_qitem(a, tb, g, id, &it, tile_rows, tile_first); id += workers) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(acc_full + buf, acc_phase, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const int r_local = q * 32 + lane;
            const int64_t n = (int64_t)it.n0 + r_local;             // this lane's output column
            const bool mine = r_local < a.rows_w && n < a.N;
            const int chunks = q * 32 < a.rows_w ? (it.tokens + 31) >> 5 : 0;
            auto release_acc = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) mbar_arrive_cluster(leader_base + (smem_u32(acc_empty + buf) - own_base));
                    else mbar_arrive(acc_empty + buf);
                }
            };
            if (e >= chunks) release_acc();              // nothing to drain for this warp
            const uint32_t acc = tmem_base + buf * (uint32_t)a.tok_cap + ((uint32_t)(q * 32) << 16);
            if (!pair_ok) {                              // odd N: two-byte stores, chunk by chunk
#pragma unroll 1
                for (int c = e; c < chunks; c += 2) {
                    uint32_t r[32];
                    tmem_ld32(acc + (uint32_t)(c * 32), r);
                    tmem_ld_wait();
                    if (c + 2 >= chunks) release_acc();
                    const int left = mine ? it.tokens - c * 32 : 0;
                    uint16_t* p = a.out + (int64_t)(it.row0 + c * 32) * a.N + n;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (j < left) *p = f32_to_bf16_bits(__uint_as_float(r[j]));
                        p += a.N;
                    }
                }
                if (++buf == (uint32_t)a.acc_bufs) { buf = 0; acc_phase ^= 1; }
                continue;
            }
            // everything this warp drains is packed into registers first, so that the accumulator is free for the next
            // item before the stores begin: word i of chunk c = tokens 32c + 2i, 2i + 1 of this lane's column
            uint32_t v[kQEpiChunks][16];
#pragma unroll
            for (int k = 0; k < kQEpiChunks; ++k) {
                if (e + 2 * k >= chunks) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t r[16];
                    tmem_ld16(acc + (uint32_t)((e + 2 * k) * 32 + h * 16), r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[k][8 * h + j] = pack_bf16x2(__uint_as_float(r[2 * j + 1]), __uint_as_float(r[2 * j]));
                }
            }
            if (e < chunks) release_acc();
            // lanes 2i and 2i+1 swap words: the even lane stores columns (n, n+1) of token 2j, the odd lane (n-1, n) of
            // token 2j+1 -- 4-byte stores, 64 bytes per half warp
            const int odd = lane & 1;
            const uint32_t pick = odd ? 0x3276u : 0x5410u;       // (got.hi, own.hi) or (own.lo, got.lo)
            uint16_t* p = a.out + (int64_t)(it.row0 + e * 32 + odd) * a.N + (n - odd);
            const int64_t step = 2 * a.N;
            int left = mine ? it.tokens - e * 32 - odd : 0;      // store while 2j < left
#pragma unroll
            for (int k = 0; k < kQEpiChunks; ++k) {
                if (e + 2 * k >= chunks) break;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, v[k][j], 1);
                    if (2 * j < left) *reinterpret_cast<uint32_t*>(p) = prmt(v[k][j], got, pick);
                    p += step;
                }
                p += 16 * step;                                  // the other warp's chunk
                left -= 64;
            }
            if (++buf == (uint32_t)a.acc_bufs) { buf = 0; acc_phase ^= 1; }
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before();
    // in a pair neither CTA may free its tensor memory or leave while the other's MMAs and arrivals can reach it
    if (CG == 2) cluster_sync_all();
    else __syncthreads();
    if (*abort_flag) {               // a wait gave up: give the copies in flight time to land before the memory goes
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) {
        }
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (CG == 2) tmem_dealloc_2(tmem_base, kQTmemCols);
        else tmem_dealloc(tmem_base, kQTmemCols);
    }
    if (threadIdx.x == 0 && *abort_flag && a.status) atomicOr(a.status, GNF4B_ST_TIMEOUT);
}

// CTA pairs: where a group is long and an item has enough stages to pay for handing it over between two CTAs.  A box row of
// 128 bytes is one line of L2 where rows start on 128-byte lines (K a multiple of 256) and two where they do not; single CTAs
// are held up by the second line, and there pairs win on every long group.  On the lines the two are about even, and
// pairs fall behind where the last span of scales holds one or two stages (K = 1280, 1536, 2304).
// Microseconds of pairs / of single CTAs, 32 experts, N = 4096, equal groups:
//                  300 rows    384         448         512         1024
//   off:  K = 736   49 / 45    51 / 48     54 / 53     57 / 55    105 / 100
//             1056  64 / 60    67 / 64     70 / 72     72 / 75    122 / 135
//             1312  67 / 66    71 / 70     73 / 80     76 / 83    132 / 153
//             2080  94 / 86    94 / 92     97 / 106   100 / 111   183 / 210
//             2880  95 / 90   100 / 101   105 / 113   111 / 119   205 / 227
//             2912 100 / 119  108 / 119   115 / 139   122 / 142   232 / 275
//             4128 148 / 156  156 / 167   166 / 192   180 / 204   351 / 391
//             7200 248 / 249  256 / 267   273 / 311   298 / 326   592 / 627
//   on:   K = 1024  42 / 39    44 / 42     48 / 46     50 / 49     93 / 93
//             1536  61 / 52    64 / 58     66 / 63     69 / 68    124 / 125
//             1792  64 / 58    68 / 66     72 / 72     76 / 77    137 / 144
//             2048  65 / 62    70 / 69     75 / 75     79 / 81    143 / 150
//             2304  89 / 73    93 / 81     95 / 89    100 / 95    181 / 174
//             2816  93 / 82    96 / 91    101 / 100   107 / 106   196 / 198
//             4096 125 / 109  127 / 120   130 / 131   137 / 137   256 / 261
//             7168 220 / 177  207 / 192   213 / 208   223 / 221   415 / 432
// Off the lines at 416 rows: N = 5760, K = 2880 144 / 152 (384 rows: 137 / 140); 64 experts, N = 2048, K = 1312 74 / 91 (72 / 80);
// 16 experts, N = 4096, K = 2080 66 / 64 (59 / 58); 8 experts, N = 14336, K = 4128 185 / 173 (193 / 154).  K = 1056 with 576
// rows 98 / 89.  On them: 128 experts, N = 1536, K = 2048, 1024 rows 219 / 234; 16 experts, N = 4096, K = 7168 213 / 207.
constexpr int kQPairRows = 400, kQPairRowsAligned = 448;
constexpr int kQPairStages = 6;                                        // off the lines: K > 1280
constexpr int kQPairStagesAlignedLo = 7, kQPairStagesAlignedHi = 8;    // on them: 1536 < K <= 2048

struct W4A4Plan {
    int rows_w, tok_cap, xbox, x_bytes, x_blocks, stages, acc_bufs;
    int pair;           // CTA pairs
    size_t smem;
};

// Tile shape from the row counts alone.  max_rows <= 0: unknown, any group may be long.  Fewer than two stages: the device
// has too little shared memory.
static inline W4A4Plan w4a4_plan(int64_t T, int32_t G, int64_t N, int64_t K, int32_t max_rows, int sm_count, int smem_optin) {
    W4A4Plan p;
    const int64_t longest = max_rows > 0 ? (max_rows < T ? max_rows : T) : T;
    p.tok_cap = (int)round_up(longest < 256 ? longest : 256, 16);
    p.xbox = p.tok_cap <= 16 ? 16 : p.tok_cap <= 64 ? 32 : 64;
    p.x_bytes = (int)round_up(p.tok_cap, p.xbox) * kQRowBytes;
    p.x_blocks = (p.tok_cap + 127) / 128;
    p.rows_w = 128;
    if (longest <= 64) {
        // streaming weights: the tile height that shares the rows out most evenly; an item costs its bytes and, for
        // hand-overs between the roles, about as much time as 9000 bytes more
        double best = 1e30;
        for (int r = 128; r >= 64; r -= 8) {
            const int64_t rounds = ceil_div((int64_t)G * ceil_div(N, r), sm_count);
            const double cost = (double)rounds * ((double)r * (double)K * (17.0 / 32.0) + 9000.0);
            if (cost < best) { best = cost; p.rows_w = r; }
        }
    }
    const int64_t k_stages = ceil_div(K, kQStageK);
    const bool on_lines = (K / 2) % 128 == 0;
    p.pair = on_lines ? longest >= kQPairRowsAligned && k_stages >= kQPairStagesAlignedLo && k_stages <= kQPairStagesAlignedHi
                      : longest >= kQPairRows && k_stages >= kQPairStages;
    if (p.pair) {
        p.tok_cap = (int)round_up(p.tok_cap, 32);
        p.xbox = 64;
        p.x_bytes = (int)round_up(p.tok_cap / 2, p.xbox) * kQRowBytes;
    }
    const size_t fixed = w4a4_fixed_bytes(p.x_blocks), room = (size_t)smem_optin > fixed ? (size_t)smem_optin - fixed : 0;
    p.stages = (int)(room / (size_t)(kQWTile + p.x_bytes));
    if (p.stages > kQMaxStages) p.stages = kQMaxStages;
    p.acc_bufs = 2 * p.tok_cap + p.stages * 8 * (1 + p.x_blocks) <= kQTmemCols ? 2 : 1;
    p.smem = fixed + (size_t)p.stages * (kQWTile + p.x_bytes);
    return p;
}

}  // namespace gnf4b
