// k_kv8_attention.cu -- attention of Q rows over the paged 8-bit cache.
//
//   s_j = scale q.k_j,  out = sum_j p_j v_j,  p = softmax(s),  k_j = code * page scale
//
// A block holds 8 or 16 rows of one sequence and k/v head: (query token, head
// of the group) pairs, token-major.  The blocks' keys, in tiles of 128 and in
// one order, are cut into equal shares, one for each CTA that fits on the
// device: lengths are on the device and often uneven, and equal shares of them
// leave no CTA waiting for a long sequence and write few partial results (at
// most two a CTA, whatever the batch).  A CTA walks through its share block by
// block; a second kernel joins the blocks that a cut went through.
//
// Within a CTA each of 4 warps takes every fourth step of 32 keys (16 for heads
// over 128) through a ring of TMA stages of its own: one lane issues the copies,
// and no barrier of the CTA is in the loop.
//   S^T = K Q^T, ldmatrix the codes' registers: int8 codes as they are
//     (m16n8k32, Q as three digits: an 8-bit product costs half an f16 one, the
//     codes' conversion more than all of them), e4m3 codes as f16 (QParts);
//   O^T = V^T P^T, m16n8k16 on f16: S^T's registers, transposed 8 x 8, are P^T's
//     operands; lane (g, t) (g = lane / 4, t = lane % 4) holds elements 16 g ..
//     16 g + 15 (of 128) of keys 2t, 2t + 1, 2t + 8 and 2t + 9 with 16-byte
//     loads, and pairs and converts them.
// TMA's swizzle (the 16-byte piece c of key r lies at c ^ (r & 7)) puts the 8
// rows of an ldmatrix and the 8 lanes of a 16-byte access into different banks.
//
// Precision.  A row of q is held to 2^-22 of its largest element or better,
// products and their sums are exact (int8) or f32.  Weights p are f16 relative
// to a power of two near the row's largest (half a step 2^-12, an eighth of the
// bf16 output's), for f32 rows two f16 (hi + lo).  Sums, maxima and the sum of p
// are f32.  The values' scale joins the exponent, p v_scale = 2^(s + log2 v_scale
// - r'), with a reference r' of its own per row, so pages of any scales keep
// their weight.  References are whole numbers and move only when a score passes
// them by 2^4: rescaling is rare, by ex2.approx (2^-22) of a whole number.  A weight
// more than 2^-25 below the row's largest is an f16 subnormal, off by at most 2^-36 of
// the largest.
//
// What bounds it and what it measured (8 k/v heads): the codes' bytes where there
// are many keys a row, 64 sequences of 1 .. 8191 keys, 64 heads of 128, int8, 95 us,
// 5.7 TB/s (a copy: 6.5), one of 131071, e4m3, 56 us, 4.8 TB/s, of it 15 us above the
// bytes' time: launch, shares, table -> scale -> codes -> products, join.
// With 16 rows a block and heads of 64 (48 sequences, 1 .. 8 tokens, 32 heads, a
// window of 1000) the warps' instructions, about 550 for 32 keys and 1800 a block,
// issued at half rate by the 12 warps that registers allow: 34 us.
#include "kv8_mma.cuh"
#include "phases.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTileKeys = 128;     // keys that shares are counted in
constexpr int kLeastTiles = 2;     // tiles below which a share is not cut further
// What a block costs besides its keys, in tiles (64 sequences of up to 8191 keys
// at 2: 103 us, 4: 95, 6: 97).
constexpr int kHeadTiles = 4;
constexpr int kMostCtas = 1024;
constexpr float kSlack = 4.0f;     // how far (log2) scores may pass a reference
constexpr float kLift = 11.0f;     // weights are held times 2^11: up to 2^15 in f16
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoRef = -3.0e38f;  // the reference of a row that has seen no key

// The first cut through a block: what the joining kernel needs.
struct alignas(16) Cut {
    int parts;  // 0: the share begins with a block, or the block was cut before
    int lone;   // where the first part is; the others are the following CTAs' first
    int rows, at, lo, head;  // the block's live rows, its first one in the sequence's
                             // (token, head of the group) rows, those' first token
    int unused[2];
};

// Where CTA c's share begins.
__device__ __forceinline__ int64_t share(int64_t each, int rest, int c) {
    return c * each + min(c, rest);
}
// a / b of a >= 0, b > 0, in 32 bits where that does.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

struct Args {
    CUtensorMap k_map, v_map;  // [n_pages * n_kv_heads][page][d] codes
    kv8::Batch b;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride;
    const float *k_scale, *v_scale;
    unsigned* status;
    Cut* cuts;      // [CTA] the block that its share begins inside
    float* part;    // [CTA][2][block_rows][d] its first and last block's partial outputs
    float2* state;  // [CTA][2][block_rows] a row's (reference, sum)
    float scale;
    int hq, hkv, d, window, max_rows, max_len, block_rows, whole, vec, vec_out;
};

// A sequence's blocks and the tiles that its longest one may have.
struct Load {
    kv8::Seq s;
    bool ok;  // within the call's bounds
    int blocks, tiles;
    // A block spans kHeadTiles, which stand for its fixed cost and are not cut,
    // and its tiles.
    __device__ int span() const { return kHeadTiles + tiles; }
    __device__ int64_t total(const Args& a) const { return (int64_t)blocks * a.hkv * span(); }
};

__device__ __forceinline__ Load load_of(const Args& a, int seq) {
    Load l;
    l.s = kv8::sequence(a.b, seq);
    const int group = a.hq / a.hkv;
    l.ok = l.s.len <= a.max_len && l.s.n <= a.max_rows &&
           l.s.len <= ((int64_t)a.b.width << a.b.page_shift);
    l.blocks = (l.s.n * group + a.block_rows - 1) / a.block_rows;  // rows * group fits an int
    int64_t keys = l.ok ? l.s.len : 0;
    // a block's tokens span (block_rows - 1) / group + 1 positions at most, and its
    // first step begins up to 31 keys early
    if (a.window) keys = min(keys, (int64_t)a.window + (a.block_rows - 1) / group + 32);
    l.tiles = a.whole ? 1 : max(1, (int)((keys + kTileKeys - 1) / kTileKeys));
    return l;
}

// What a block of rows attends.
struct Block {
    int rows;       // live rows of the block
    int from, end;  // keys [from, end), from a whole step
    int seen;       // the first key that a row attends: those from `from` to it are masked
};

__device__ __forceinline__ Block block_of(const Args& a, const Load& l, int block) {
    Block k;
    const int group = a.hq / a.hkv, at = block * a.block_rows;
    k.rows = min(a.block_rows, l.s.n * group - at);
    k.from = k.end = k.seen = 0;
    if (l.ok) {
        const int p0 = l.s.first + at / group, p1 = l.s.first + (at + k.rows - 1) / group;
        k.end = max(p1 + 1, 0);
        k.seen = min(kv8::first_seen(p0, a.window), k.end);
        k.from = k.seen & ~31;
    }
    return k;
}

// Where the 16-byte piece c of a key lies in a tile of KEYS keys: DP = 64 has
// rows of 64 bytes and that swizzle, DP = 256 two tiles of 128-byte rows.
template <int DP, int KEYS>
__device__ __forceinline__ int place(int key, int c) {
    if constexpr (DP == 64) return key * 64 + (c ^ (key >> 1 & 3)) * 16;
    return (c >> 3) * KEYS * 128 + key * 128 + ((c ^ key) & 7) * 16;
}

// CTAs per SM: what registers (O: DP NB / 4 a lane) and shared memory allow.
constexpr int ctas_of(int dp, int nb, bool f32) {
    return dp * nb >= (f32 ? 128 : 256) ? 2 : dp * nb >= (f32 ? 64 : 128) ? 3 : 4;
}
inline int ctas_per_sm(int d, int block_rows, bool f32) {
    return ctas_of(d <= 64 ? 64 : d <= 128 ? 128 : 256, block_rows / 8, f32);
}

// Shapes of a kernel for heads of up to DP elements and blocks of 8 NB rows.
template <typename T, int FORMAT, int DP, int NB>
struct Shape {
    static constexpr bool kSplit = sizeof(T) == 4;  // hi + lo weights
    static constexpr int kKeys = DP == 256 ? 16 : 32;  // a warp's step
    static constexpr int kHalves = kKeys / 16;
    static constexpr int kStages = DP == 128 ? 2 : 3;
    static constexpr int kStageBytes = 2 * kKeys * DP;
    static constexpr int kWords = DP / 16;  // words of four elements a lane has of a row of q
    static constexpr int kRows = 8 * NB;
    // Q's operands stay in registers when they are few
    static constexpr int kQPairs = kv8::QParts<T, FORMAT>::kRegs * kWords / 2;
    static constexpr bool kQReg = kQPairs * NB <= 16;
    static constexpr int kQBytes = kQPairs * NB * 256;
    static constexpr int kRing = kWarps * kStages * kStageBytes;  // a multiple of 1024
    static constexpr int kPitch = DP == 64 ? DP + 2 : DP + 4;  // floats of a row's state
    static constexpr int kJoin = kWarps * kRows * (kPitch + 4) * 4;
    static constexpr int kBytes =
        (kRing > kJoin ? kRing : kJoin) + kQBytes + 1024;  // 1024: to align
    static constexpr int kCtas = ctas_of(DP, NB, kSplit);
};

// (sum up to this thread, sum over the block) of v.
__device__ __forceinline__ longlong2 block_scan(int64_t v, int64_t* warps) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(tbk::kFull, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int64_t all = 0, before = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += warps[i];
        all += warps[i];
    }
    return make_longlong2(before + v, all);
}

template <typename T, int FORMAT, int DP, int NB>
__global__ void __launch_bounds__(kThreads, Shape<T, FORMAT, DP, NB>::kCtas)
k_attend(const __grid_constant__ Args a) {
    using H = Shape<T, FORMAT, DP, NB>;
    using Q = kv8::QParts<T, FORMAT>;
    constexpr bool kSplit = H::kSplit, kQReg = H::kQReg;
    constexpr int kStages = H::kStages, kRows = H::kRows, kKeys = H::kKeys;
    constexpr int kHalves = H::kHalves, kQPairs = H::kQPairs, kWords = H::kWords;
    constexpr int kStride = kWarps * kKeys;  // from one of a warp's steps to its next
    constexpr int kTiles = DP / 16;          // 16-wide output tiles
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[kWarps * kStages];
    __shared__ int64_t scan[kWarps], found_begin;
    __shared__ int found_seq;
    __shared__ uint4 top_s[kRows];
    // TMA's swizzle goes by the address: tiles start on 1024 bytes
    uint8_t* smem = smem_raw + (-tbk::smem_addr(smem_raw) & 1023u);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.hq / a.hkv;
    uint8_t* ring = smem + warp * kStages * H::kStageBytes;
    uint64_t* bar = bars + warp * kStages;
    if (threadIdx.x == 0) {
        kv8::prefetch_map(&a.k_map);
        kv8::prefetch_map(&a.v_map);
    }
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kStages; ++i) tbk::mbar_init(bar + i, 1);
        tbk::fence_mbar_init();
    }
    tbk::Phases phases;  // of each stage's barrier: a page out of range has no copy

    // This CTA's share: [tile, stop) of the batch's spans, the first in sequence
    // seq, whose own begin at seq_begin.
    int64_t tile, stop, seq_begin = 0, each;
    int seq, rest;
    {
        const int tid = threadIdx.x, n_seqs = a.b.n_seqs;
        int64_t w = tid < n_seqs ? load_of(a, tid).total(a) : 0, tiles = w;
        for (int i = tid + kThreads; i < n_seqs; i += kThreads) tiles += load_of(a, i).total(a);
        longlong2 sum = block_scan(tiles, scan);  // (up to this thread, all)
        tiles = sum.y;
        const int64_t want = a.whole ? quotient(tiles, kHeadTiles + 1)
                                     : (tiles + kLeastTiles - 1) / kLeastTiles;
        const int ctas = (int)min((int64_t)gridDim.x, want);
        if (tid == 0 && a.cuts) a.cuts[blockIdx.x].parts = 0;
        if ((int)blockIdx.x >= ctas) return;
        each = quotient(tiles, ctas);
        rest = (int)(tiles - each * ctas);
        tile = share(each, rest, blockIdx.x);
        stop = share(each, rest, blockIdx.x + 1);
        if (n_seqs > kThreads) sum = block_scan(w, scan);
        for (int i = tid;;) {  // ends: the sum over all is above tile
            if (tile >= seq_begin + sum.x - w && tile < seq_begin + sum.x) {
                found_seq = i;
                found_begin = seq_begin + sum.x - w;
            }
            __syncthreads();
            if (tile < seq_begin + sum.y) break;
            seq_begin += sum.y;
            i += kThreads;
            w = i < n_seqs ? load_of(a, i).total(a) : 0;
            sum = block_scan(w, scan);
        }
        seq = found_seq;
        seq_begin = found_begin;
    }
    // the joining kernel may take its place on the SMs as CTAs end
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Load load = load_of(a, seq);

    for (bool first_block = true; tile < stop; first_block = false) {
        while (tile >= seq_begin + load.total(a)) {
            seq_begin += load.total(a);
            load = load_of(a, ++seq);
        }
        const int in_seq = (int)quotient(tile - seq_begin, load.span());
        const int head = in_seq / load.blocks, block = in_seq - head * load.blocks;
        const int64_t unit_begin = seq_begin + (int64_t)in_seq * load.span();
        // a share that ends within a block's head leaves it all to the next CTA
        if (stop - unit_begin <= kHeadTiles) break;
        const int skip = max(0, (int)(tile - unit_begin) - kHeadTiles);
        const int till = (int)min((int64_t)load.tiles, stop - unit_begin - kHeadTiles);
        tile = unit_begin + kHeadTiles + till;
        const bool whole = skip == 0 && till == load.tiles;
        const Block blk = block_of(a, load, block);
        if (threadIdx.x == 0) {
            const int64_t before = share(each, rest, blockIdx.x - 1);
            if (first_block && skip > 0 && before <= unit_begin + kHeadTiles) {
                // the last CTA whose share begins before the block's end
                const int64_t end = unit_begin + load.span() - 1, longer = rest * (each + 1);
                const int last = (int)(end < longer ? quotient(end, each + 1)
                                                    : rest + quotient(end - longer, each));
                a.cuts[blockIdx.x] = {last - (int)blockIdx.x + 2,
                                      2 * ((int)blockIdx.x - 1) + (before < unit_begin),
                                      blk.rows, block * kRows, load.s.lo, head, {}};
            }
            if (!load.ok) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
        }
        const int begin = blk.from + skip * kTileKeys;
        const int end = a.whole ? blk.end
                                : (int)min(blk.from + (int64_t)till * kTileKeys, (int64_t)blk.end);

        // Q: row 8 b + g of the block, words of elements 16 j + 4 t .. + 3, those
        // with j % 4 = warp; asked for first, used when the copies are on their way
        constexpr int kMine = kWords / kWarps;
        float x[NB][kMine][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int i = 8 * b + g;
            const bool live = i < blk.rows;
            const int at = block * kRows + i, tok = live ? at / group : 0;
            const int hh = live ? at - tok * group : 0;
            const T* q = static_cast<const T*>(a.q) + (load.s.lo + tok) * a.q_stride +
                         (int64_t)(head * group + hh) * a.d;
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                const int word = 16 * (warp + kWarps * j);
                kv8::load4(q + word + 4 * t, live && word < a.d, a.vec, x[b][j]);
            }
        }

        // the warp's steps: keys first + kStride n .. + kKeys - 1
        const int first = begin + warp * kKeys;
        const int n_steps = end > first ? (end - first + kStride - 1) / kStride : 0;
        const int32_t* table = a.b.table + seq * a.b.table_stride;
        // A step's 16-key halves are in one page, or, with pages of 16, in two.
        const bool one_page = a.b.page_shift >= 5;
        const int in_page = one_page ? kKeys : 16;  // keys that a lookup is for
        auto page_of = [&](int i) {  // the page of half-step i, -1 if it has none
            const int key =
                first + i / kHalves * kStride + (kHalves == 2 && !one_page ? i % 2 * 16 : 0);
            // (a page all in front of a window may be gone)
            if (i / kHalves >= n_steps || key >= end || key + in_page <= blk.seen) return -1;
            const int id = table[key >> a.b.page_shift];
            if (id >= 0 && id < a.b.n_pages) return id;
            atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
            return -1;
        };
        // Lane i has the page of half-step 32 m + i and its scales, m the batch
        // that is being issued; the next batch's pages are on their way.
        constexpr int kBatch = 32 / kHalves;  // steps
        int ids = page_of(lane), ids_next = page_of(32 + lane);
        float ks_issued = 0.0f, vs_issued = 0.0f, ks = 0.0f, vs = 0.0f;
        uint32_t pages_issued, pages = 0;  // which half-steps of the batch have a page
        auto load_scales = [&] {
            pages_issued = __ballot_sync(tbk::kFull, ids >= 0);
            if (ids >= 0) {
                const int unit = ids * a.hkv + head;
                ks_issued = a.k_scale[unit];
                vs_issued = a.v_scale[unit];
            }
        };
        load_scales();
        auto issue = [&](int n, int stage) {
            const int i = n % kBatch * kHalves;
            if (i == 0 && n > 0) {
                ids = ids_next;
                load_scales();
                ids_next = page_of(n * kHalves + 32 + lane);
            }
            const int id0 = __shfl_sync(tbk::kFull, ids, i);
            const int id1 = kHalves == 2 ? __shfl_sync(tbk::kFull, ids, i + 1) : -1;
            if (lane == 0 && (id0 >= 0 || id1 >= 0)) {
                uint8_t* dst = ring + stage * H::kStageBytes;
                const int slot = (first + n * kStride) & ((1 << a.b.page_shift) - 1);
                auto copy = [&](int id, int at, int slot) {  // a box, from the stage's key `at`
#pragma unroll
                    for (int h = 0; h < (DP + 127) / 128; ++h) {
                        uint8_t* d = dst + h * kKeys * 128 + at * (DP < 128 ? DP : 128);
                        kv8::tma_load3(d, &a.k_map, h * 128, slot, id * a.hkv + head, bar + stage);
                        kv8::tma_load3(d + kKeys * DP, &a.v_map, h * 128, slot, id * a.hkv + head,
                                       bar + stage);
                    }
                };
                if (kHalves == 1 || one_page) {
                    tbk::mbar_expect_tx(bar + stage, H::kStageBytes);
                    copy(id0, 0, slot);
                } else {
                    tbk::mbar_expect_tx(bar + stage,
                                        ((id0 >= 0) + (id1 >= 0)) * (H::kStageBytes / 2));
                    if (id0 >= 0) copy(id0, 0, slot);
                    if (id1 >= 0) copy(id1, 16, 0);
                }
            }
        };
#pragma unroll
        for (int n = 0; n < kStages - 1; ++n) issue(n, n);

        // Each warp splits its quarter of Q; a row's sums of products are multiplied
        // with qf, but for the page's scale.  A row with a NaN or an infinity (whose
        // bits are the largest) is NaN.
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < kMine; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(x[b][j][e])));
            top = max(top, __shfl_xor_sync(tbk::kFull, top, 1));
            top = max(top, __shfl_xor_sync(tbk::kFull, top, 2));
            if (t == 0) reinterpret_cast<uint32_t*>(top_s)[(8 * b + g) * 4 + warp] = top;
        }
        __syncthreads();
        uint32_t* qs = reinterpret_cast<uint32_t*>(smem + H::kBytes - 1024 - H::kQBytes);
        const uint2* q2 = reinterpret_cast<const uint2*>(qs) + lane;
        float qf[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint4 u = top_s[8 * b + g];
            const float top = __uint_as_float(max(max(u.x, u.y), max(u.z, u.w)));
            const Q parts(top < INFINITY ? top : 0.0f);
            qf[b] = top < INFINITY ? parts.unit * (a.scale * kLog2e) : NAN;
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                uint32_t w[Q::kRegs];
                parts.split(x[b][j], w);
                // pairs of registers: int8 of two words, e4m3 of one
                const int word = warp + kWarps * j;
#pragma unroll
                for (int p = 0; p < Q::kRegs; ++p) {
                    const int at = FORMAT == kv8::kInt8 ? p * kWords + word
                                                        : (p / 2 * kWords + word) * 2 + p % 2;
                    qs[((at / 2 * NB + b) * 32 + lane) * 2 + at % 2] = w[p];
                }
            }
        }
        // S^T's columns: rows 8 b + 2 t + e, keys [see_lo, see_hi] each
        float qc[NB][2];
        int see_lo[NB][2], see_hi[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                qc[b][e] = __shfl_sync(tbk::kFull, qf[b], (2 * t + e) * 4);
                const int i = 8 * b + 2 * t + e;
                // rows of the block that are not there see all and are not stored
                const bool live = i < blk.rows;
                const int p = load.s.first + (block * kRows + i) / group;
                see_hi[b][e] = live ? p : INT32_MAX;
                see_lo[b][e] = live ? kv8::first_seen(p, a.window) : 0;
            }
        __syncthreads();
        uint2 qr[kQReg ? kQPairs : 1][NB];
        if constexpr (kQReg) {
#pragma unroll
            for (int i = 0; i < kQPairs; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) qr[i][b] = q2[(i * NB + b) * 32];
        }
        auto q_pair = [&](int i, int b) {
            if constexpr (kQReg)
                return qr[i][b];
            else
                return q2[(i * NB + b) * 32];
        };

        float o[kTiles][NB][4];
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][b][e] = 0.0f;
        float ref[NB][2], vref[NB][2], sum[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                ref[b][e] = vref[b][e] = kNoRef;
                sum[b][e] = 0.0f;
            }

        int at_stage = kStages - 1;
        bool lost = false;  // a copy did not come
        auto copy_came = [&](int i) {
            return phases.wait(i, [&](uint32_t parity) {
                return __all_sync(tbk::kFull, tbk::mbar_wait(bar + i, parity, a.status));
            });
        };
        for (int n = 0; n < n_steps; ++n) {
            const int i0 = n % kBatch * kHalves;
            if (i0 == 0) {
                ks = ks_issued;
                vs = vs_issued;
                pages = pages_issued;
            }
            __syncwarp();  // step n - 1's stage has been read: it is the next to be filled
            issue(n + kStages - 1, at_stage);
            at_stage = at_stage == kStages - 1 ? 0 : at_stage + 1;
            const uint32_t have = pages >> i0 & ((1 << kHalves) - 1);
            if (have == 0) continue;
            float k_scale[kHalves], lv[kHalves];  // the values' scale as an exponent
#pragma unroll
            for (int f = 0; f < kHalves; ++f) {
                k_scale[f] = __shfl_sync(tbk::kFull, ks, i0 + f);
                const float v_scale = __shfl_sync(tbk::kFull, vs, i0 + f);
                lv[f] = (float)((int)(__float_as_uint(v_scale) >> 23) - 127);
            }
            uint8_t* stage = ring + at_stage * H::kStageBytes;
            if (!copy_came(at_stage)) {
                // the output is invalid and flagged.  No copy may be in flight when the
                // CTA ends: wait for this one and those behind it, bounded.
                for (int i = 0; i < kStages; ++i)
                    if (page_of((n + i) * kHalves) >= 0 ||
                        (kHalves == 2 && page_of((n + i) * kHalves + 1) >= 0))
                        copy_came((at_stage + i) % kStages);
                lost = true;
                break;
            }
            const int key0 = first + n * kStride;
            uint8_t* values = stage + kKeys * DP;
            const uint32_t stage_s = tbk::smem_addr(stage);
            const bool gaps = key0 < blk.seen || key0 + kKeys > blk.end ||
                              have != (1 << kHalves) - 1;
            if (gaps) {
                // slots that no row of the block attends, or of no page, may hold anything,
                // NaN codes too: a weight of zero needs a finite value beside it
                for (int i = lane; i < kKeys * DP / 16; i += 32) {
                    const int key = i % kKeys;
                    if (key0 + key < blk.seen || key0 + key >= blk.end || !(have >> key / 16 & 1))
                        *reinterpret_cast<uint4*>(values + place<DP, kKeys>(key, i / kKeys)) =
                            make_uint4(0, 0, 0, 0);
                }
                tbk::fence_proxy_async_shared();  // the stage is filled by TMA again
                __syncwarp();
            }

            // S^T in log2 units: s[f][b][2 i + e] is key key0 + 16 f + g + 8 i, row
            // 8 b + 2 t + e
            float s[kHalves][NB][4];
#pragma unroll
            for (int f = 0; f < kHalves; ++f) {
                uint32_t w[kWords / 2][4];
#pragma unroll
                for (int j = 0; j < kWords / 2; ++j)
                    kv8::load_operand(stage_s + place<DP, kKeys>(16 * f + lane % 16, 2 * j + lane / 16),
                                      w[j]);
                if constexpr (FORMAT == kv8::kInt8) {
                    // whole sums below 2^22 over the bits of 1.5 * 2^23 are that f32
                    // plus the sum
                    constexpr int kBits = 0x4b400000;
                    constexpr float kBase = 12582912.0f;
                    const int base[4] = {kBits, kBits, kBits, kBits};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        int d[3][4];
#pragma unroll
                        for (int p = 0; p < 3; ++p)
#pragma unroll
                            for (int j = 0; j < kWords / 2; ++j) {
                                const uint2 q = q_pair(p * kWords / 2 + j, b);
                                if (j == 0)
                                    kv8::mma_codes(d[p], w[j], q.x, q.y, base);
                                else
                                    kv8::mma_codes(d[p], w[j], q.x, q.y, d[p]);
                            }
                        float(&z)[4] = s[f][b];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            z[e] = fmaf(__int_as_float(d[0][e]), 16384.0f, -kBase * 16384.0f);
                            z[e] = fmaf(__int_as_float(d[1][e]) - kBase, 128.0f, z[e]);
                            z[e] += __int_as_float(d[2][e]) - kBase;
                        }
                    }
                } else {
                    // a word's elements 0, 1 are the operand's 2t, 2t + 1 and its 2, 3
                    // 2t + 8, 2t + 9, as q's pairs have them
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[f][b][e] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        const uint32_t k0 = w[j / 2][j % 2 * 2], k1 = w[j / 2][j % 2 * 2 + 1];
                        const uint32_t a0 = kv8::e4m3_pair(k0, false), a1 = kv8::e4m3_pair(k1, false);
                        const uint32_t a2 = kv8::e4m3_pair(k0, true), a3 = kv8::e4m3_pair(k1, true);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int p = 0; p < Q::kParts; ++p) {
                                const uint2 q = q_pair(p * kWords + j, b);
                                kv8::mma_f16(s[f][b], a0, a1, a2, a3, q.x, q.y);
                            }
                    }
                }
            }
            bool inside = !gaps, over = false;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    inside &= key0 >= see_lo[b][e] && key0 + kKeys - 1 <= see_hi[b][e];
#pragma unroll
                    for (int f = 0; f < kHalves; ++f) {
                        const float scale = qc[b][e] * k_scale[f];
                        s[f][b][e] *= scale;
                        s[f][b][2 + e] *= scale;
                    }
                }
            if (!__all_sync(tbk::kFull, inside)) {
#pragma unroll
                for (int f = 0; f < kHalves; ++f)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = key0 + 16 * f + g + 8 * (i >> 1);
                            if (j < see_lo[b][i & 1] || j > see_hi[b][i & 1] || !(have >> f & 1))
                                s[f][b][i] = -INFINITY;
                        }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int f = 0; f < kHalves; ++f) {
                        const float hi = fmaxf(s[f][b][e], s[f][b][2 + e]);
                        over |= hi > ref[b][e] + kSlack || hi + lv[f] > vref[b][e] + kSlack;
                    }
            if (__any_sync(tbk::kFull, over)) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float hi = -INFINITY, hv = -INFINITY;
#pragma unroll
                        for (int f = 0; f < kHalves; ++f) {
                            const float x = fmaxf(s[f][b][e], s[f][b][2 + e]);
                            hi = fmaxf(hi, x);
                            hv = fmaxf(hv, ceilf(x) + lv[f]);
                        }
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) {
                            hi = fmaxf(hi, __shfl_xor_sync(tbk::kFull, hi, x));
                            hv = fmaxf(hv, __shfl_xor_sync(tbk::kFull, hv, x));
                        }
                        const float m = fmaxf(ref[b][e], ceilf(hi)), mv = fmaxf(vref[b][e], hv);
                        if (m > ref[b][e]) sum[b][e] *= kv8::exp2_fast(ref[b][e] - m);
                        if (mv > vref[b][e]) {
                            const float keep = kv8::exp2_fast(vref[b][e] - mv);
#pragma unroll
                            for (int i = 0; i < kTiles; ++i) {
                                o[i][b][e] *= keep;
                                o[i][b][2 + e] *= keep;
                            }
                        }
                        ref[b][e] = m;
                        vref[b][e] = mv;
                    }
            }
#pragma unroll
            for (int f = 0; f < kHalves; ++f) {
                // weights: for the sum, and times the values' scale as P^T's operands
                uint32_t ph[NB][2], pl[NB][2];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float m = ref[b][e], mv = vref[b][e] - lv[f] - kLift;
                        sum[b][e] += kv8::exp2_fast(s[f][b][e] - m) +
                                     kv8::exp2_fast(s[f][b][2 + e] - m);
                        p[e] = kv8::exp2_fast(s[f][b][e] - mv);
                        p[2 + e] = kv8::exp2_fast(s[f][b][2 + e] - mv);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t hi = kv8::pack_f16x2(p[2 * i], p[2 * i + 1]);
                        ph[b][i] = kv8::transpose8(hi);
                        if constexpr (kSplit) {
                            const __half2 h2 = *reinterpret_cast<const __half2*>(&hi);
                            pl[b][i] = kv8::transpose8(
                                kv8::pack_f16x2(p[2 * i] - __low2float(h2),
                                                p[2 * i + 1] - __high2float(h2)));
                        }
                    }
                }
                // O^T += V^T P^T: tile rows g and g + 8 are two neighbouring elements
                constexpr int kWide = DP >= 128 ? 16 : 8;  // bytes a lane takes of a key at once
#pragma unroll
                for (int h = 0; h < (DP + 127) / 128; ++h) {
                    uint32_t w[4][kWide / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = 16 * f + 2 * t + (i & 1) + (i & 2) * 4;
                        if constexpr (DP >= 128) {
                            const uint4 x = *reinterpret_cast<const uint4*>(
                                values + place<DP, kKeys>(key, 8 * h + g));
                            w[i][0] = x.x;
                            w[i][1] = x.y;
                            w[i][2] = x.z;
                            w[i][3] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2*>(
                                values + place<DP, kKeys>(key, g >> 1) + (g & 1) * 8);
                            w[i][0] = x.x;
                            w[i][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kWide / 4; ++j) {
                        uint32_t lo[4], hi[4];
                        kv8::words<FORMAT>(w[0][j], w[1][j], lo);
                        kv8::words<FORMAT>(w[2][j], w[3][j], hi);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                float(&d)[4] = o[h * 8 + 2 * j + i][b];
                                kv8::mma_f16(d, lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1],
                                             ph[b][0], ph[b][1]);
                                if constexpr (kSplit)
                                    kv8::mma_f16(d, lo[2 * i], lo[2 * i + 1], hi[2 * i],
                                                 hi[2 * i + 1], pl[b][0], pl[b][1]);
                            }
                    }
                }
            }
        }
        // the rings are free: the warps' states meet in their place.  Where a copy was lost
        // the CTA does no more: a barrier that gave up may be in any phase
        if (__syncthreads_or(lost)) return;

        // o[h 8 + u][b][2 r + e]: element 128 h + kWide g + 2 u + r of row 8 b + 2 t
        // + e.  A row's pairs are stored turned by turn(g) within their kWide, and
        // kPitch apart, so that the lanes' pairs fall into different banks.
        constexpr int kWide = DP >= 128 ? 16 : 8;
        auto turned = [](int g, int i) {
            return kWide * g + ((i + (DP >= 128 ? g >> 1 : g >> 2) * 2) & (kWide - 1));
        };
        float* jo = reinterpret_cast<float*>(smem);
        float4* jm = reinterpret_cast<float4*>(smem + kWarps * kRows * H::kPitch * 4);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float z = sum[b][e];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(tbk::kFull, z, x);
                const int i = 8 * b + 2 * t + e;
                float* row = jo + (warp * kRows + i) * H::kPitch;
#pragma unroll
                for (int u = 0; u < kTiles; ++u)
                    *reinterpret_cast<float2*>(row + (u / 8) * 128 + turned(g, 2 * (u % 8))) =
                        make_float2(o[u][b][e], o[u][b][2 + e]);
                if (g == 0) jm[i * kWarps + warp] = make_float4(ref[b][e], vref[b][e], z, 0.0f);
            }
        __syncthreads();
        const int64_t unit = 2 * (int64_t)blockIdx.x + !first_block;
        constexpr int kPerRow = kThreads / kRows;  // threads
        const int row = threadIdx.x / kPerRow, col = threadIdx.x % kPerRow * 4;
        if (row < blk.rows) {
            float4 st[kWarps];
            float m = kNoRef, mv = kNoRef, total = 0.0f, w[kWarps];
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                st[i] = jm[row * kWarps + i];
                m = fmaxf(m, st[i].x);
                mv = fmaxf(mv, st[i].y);
            }
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                total += st[i].z * kv8::exp2_fast(st[i].x - m);
                w[i] = kv8::exp2_fast(st[i].y - mv);
            }
            const bool none = total == 0.0f;
            // O is in units of 2^(mv - lift), the sum of 2^m
            const float per = none ? 0.0f : __fdiv_rn(1.0f / 2048.0f, total) * exp2f(mv - m);
            static_assert(kLift == 11.0f, "per");
            const int at = block * kRows + row;
            const int64_t tok = load.s.lo + at / group;
            const int h = head * group + at % group;
            T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
            float* part = whole ? nullptr : a.part + (unit * kRows + row) * a.d;
#pragma unroll
            for (int i = col; i < DP; i += 4 * kPerRow) {
                if (i >= a.d) break;
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    const float* from = jo + (k * kRows + row) * H::kPitch + i / 128 * 128;
                    const int g = i % 128 / kWide;
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float2 v =
                            *reinterpret_cast<const float2*>(from + turned(g, i % kWide + e));
                        y[e] = fmaf(w[k], v.x, y[e]);
                        y[e + 1] = fmaf(w[k], v.y, y[e + 1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : y[e] * per;
                if (whole)
                    kv8::store4(out + i, a.vec_out, y);
                else
                    *reinterpret_cast<float4*>(part + i) = make_float4(y[0], y[1], y[2], y[3]);
            }
            if (col == 0) {
                if (!whole)
                    a.state[unit * kRows + row] = make_float2(m, total);
                else if (a.lse)
                    a.lse[tok * a.hq + h] =
                        none ? -INFINITY : m * 0.69314718055994531f + logf(total);
            }
        }
        // the next block's copies go where this one's states were read
        tbk::fence_proxy_async_shared();
        __syncthreads();
    }
}

// Joins the blocks that a cut went through: out = sum_c w_c out_c / sum_c w_c,
// w_c a part's sum at the largest reference.  The first cut through a block has
// CTAs for its rows; W warps a row, each with every W-th part, 8 loads in flight
// before it knows their weights, a lane four elements of 128.  What it takes is
// the chain cut -> state and part -> output and as few CTAs as do it in one go:
// four warps for every row took 8 us of 64 sequences' 102, and one warp a row 4 of
// a long sequence's 59, whose blocks have 55 parts.
constexpr int kJoinThreads = 256;
constexpr int kManyParts = 16;
template <typename T, int W>
__global__ void __launch_bounds__(kJoinThreads) k_join(const __grid_constant__ Args a) {
    constexpr int kRows = kJoinThreads / 32 / W;
    __shared__ float4 part_s[W > 1 ? kRows : 1][W][kv8::kMaxDim / 4];
    __shared__ float2 st_s[kRows][W];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group_id = warp / W, first = warp % W;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Cut cut = a.cuts[blockIdx.x + 1];
    const int row = blockIdx.y * kRows + group_id;
    if (row >= cut.rows || cut.parts == 0) return;
    const int group = a.hq / a.hkv, quads = a.d / 4;
    const int n = (cut.parts - first + W - 1) / W;  // the warp's parts
    auto unit = [&](int i) {  // of the warp's part i
        const int p = first + i * W;
        return (int64_t)(p == 0 ? cut.lone : 2 * ((int)blockIdx.x + p)) * a.block_rows + row;
    };
    const int r = cut.at + row;
    const int64_t tok = cut.lo + r / group;
    const int h = cut.head * group + r % group;
    T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
    const float4* src = reinterpret_cast<const float4*>(a.part);
    float m = kNoRef, total = 0.0f;
    for (int q = lane; q < (quads + 31) / 32 * 32; q += 32) {
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        m = kNoRef;
        total = 0.0f;
        for (int c = 0; c < n; c += 32) {
            float4 x[8];
            auto ask = [&](int i0) {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    x[u] = i0 + u < min(n, c + 32) && q < quads
                               ? __ldcg(src + unit(i0 + u) * quads + q)
                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            };
            ask(c);
            const float2 s = c + lane < n ? __ldcg(&a.state[unit(c + lane)])
                                          : make_float2(kNoRef, 0.0f);
            const float most = fmaxf(m, tbk::warp_max(s.x));
            const float keep = kv8::exp2_fast(m - most), w = s.y * kv8::exp2_fast(s.x - most);
            m = most;
            total = fmaf(total, keep, tbk::warp_sum(w));
            y = make_float4(y.x * keep, y.y * keep, y.z * keep, y.w * keep);
            for (int i0 = c; i0 < min(n, c + 32); i0 += 8) {
                if (i0 > c) ask(i0);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const float wu = __shfl_sync(tbk::kFull, w, (i0 + u - c) & 31);
                    y.x = fmaf(wu, x[u].x, y.x);
                    y.y = fmaf(wu, x[u].y, y.y);
                    y.z = fmaf(wu, x[u].z, y.z);
                    y.w = fmaf(wu, x[u].w, y.w);
                }
            }
        }
        if (W > 1) {
            part_s[group_id][first][q] = y;
        } else if (q < quads) {
            const float per[4] = {y.x, y.y, y.z, y.w};
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = total == 0.0f ? 0.0f : per[e] / total;
            kv8::store4(out + 4 * q, a.vec_out, z);
        }
    }
    if constexpr (W > 1) {
        if (lane == 0) st_s[group_id][first] = make_float2(m, total);
        asm volatile("bar.sync %0, %1;" ::"r"(group_id + 1), "n"(32 * W) : "memory");
        float w[W];
        total = 0.0f;
        m = kNoRef;
#pragma unroll
        for (int k = 0; k < W; ++k) m = fmaxf(m, st_s[group_id][k].x);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            w[k] = kv8::exp2_fast(st_s[group_id][k].x - m);
            total = fmaf(w[k], st_s[group_id][k].y, total);
        }
        for (int i = threadIdx.x % (32 * W); i < a.d; i += 32 * W) {
            float z = 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k)
                z = fmaf(w[k], reinterpret_cast<const float*>(part_s[group_id][k])[i], z);
            tbk::Elt<T>::store(out + i, total == 0.0f ? 0.0f : z / total);
        }
    }
    if (a.lse && lane == 0 && first == 0)
        a.lse[tok * a.hq + h] =
            total == 0.0f ? -INFINITY : m * 0.69314718055994531f + logf(total);
}

int check(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
          bool pointers) {
    int rc = kv8::check_cache(cache, pointers);
    if (rc == TB_OK) rc = kv8::check_batch(batch, pointers);
    if (rc != TB_OK) return rc;
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->n_heads < 1 || t->n_heads > 65535 || t->n_heads % cache->n_kv_heads ||
        t->window < 0 || t->max_rows < 0 || t->max_len < 0 || t->max_len > 1 << 30)
        return TB_ERR_INVALID_SHAPE;
    // a sequence's (token, head of the group) rows are counted in an int
    if (batch->rows * (t->n_heads / cache->n_kv_heads) > INT32_MAX / 2) return TB_ERR_INVALID_SHAPE;
    const int64_t width = (int64_t)t->n_heads * cache->head_dim;
    if (batch->rows > 1 && pointers && (t->q_stride < width || t->out_stride < width))
        return TB_ERR_INVALID_SHAPE;
    if (pointers && batch->rows && batch->n_seqs && (!t->q || !t->out || t->q == t->out))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

// How a call is laid out: rows per block, CTAs, scratch.
struct Plan {
    int block_rows, ctas, whole;
    size_t cut_bytes, part_bytes, state_bytes;
    size_t bytes() const { return cut_bytes + part_bytes + state_bytes; }
};

Plan plan_of(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
             int sm_count) {
    Plan p = {};
    const int64_t group = t->n_heads / cache->n_kv_heads;
    const int64_t rows = (t->max_rows < batch->rows ? t->max_rows : batch->rows) * group;
    // 8 rows a block where they do (64 sequences of 4000 keys, 8 heads a k/v head: 94
    // us, with blocks of 16 118), 16 where that halves the blocks
    p.block_rows = rows <= 8 ? 8 : 16;
    // at most so many blocks, of at most so many tiles
    int64_t blocks = (rows + p.block_rows - 1) / p.block_rows * batch->n_seqs;
    const int64_t most = batch->rows * group / p.block_rows + batch->n_seqs;
    blocks = (blocks < most ? blocks : most) * cache->n_kv_heads;
    int64_t keys = t->max_len;
    if (t->window && (int64_t)t->window + p.block_rows + 32 < keys)
        keys = (int64_t)t->window + p.block_rows + 32;
    const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
    p.whole = tiles <= kLeastTiles;  // blocks are not cut
    int64_t ctas =
        p.whole ? blocks : (blocks * (kHeadTiles + tiles) + kLeastTiles - 1) / kLeastTiles;
    const int64_t slots = (int64_t)sm_count * ctas_per_sm(cache->head_dim, p.block_rows, t->dtype == TB_DTYPE_F32);
    if (ctas > slots) ctas = slots;
    if (ctas > kMostCtas) ctas = kMostCtas;
    p.ctas = ctas < 1 ? 1 : (int)ctas;
    if (p.ctas == 1) p.whole = 1;
    if (!p.whole) {
        p.cut_bytes = (size_t)p.ctas * sizeof(Cut);
        p.part_bytes = (size_t)p.ctas * 2 * p.block_rows * cache->head_dim * sizeof(float);
        p.state_bytes = (size_t)p.ctas * 2 * p.block_rows * sizeof(float2);
    }
    return p;
}

template <typename T, int FORMAT, int DP, int NB>
int launch(Args& a, const TbB200Kv8* cache, dim3 grid, cudaStream_t s) {
    using H = Shape<T, FORMAT, DP, NB>;
    constexpr int bytes = H::kBytes;
    const int keys = cache->page < H::kKeys ? cache->page : H::kKeys;
    static std::atomic<uint64_t> granted{0};  // a bit per device
    int rc = kv8::once_per_device(granted, [&] {
        return cudaFuncSetAttribute(k_attend<T, FORMAT, DP, NB>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    });
    if (rc == TB_OK) rc = kv8::tile_map(&a.k_map, cache, cache->k, DP < 128 ? DP : 128, keys);
    if (rc == TB_OK) rc = kv8::tile_map(&a.v_map, cache, cache->v, DP < 128 ? DP : 128, keys);
    if (rc != TB_OK) return rc;
    k_attend<T, FORMAT, DP, NB><<<grid, kThreads, bytes, s>>>(a);
    TB_LAUNCH_CHECK("8-bit cache attention kernel");
    return TB_OK;
}

template <typename T, int FORMAT, int NB>
int launch_dim(Args& a, const TbB200Kv8* cache, dim3 grid, cudaStream_t s) {
    if (a.d <= 64) return launch<T, FORMAT, 64, NB>(a, cache, grid, s);
    if (a.d <= 128) return launch<T, FORMAT, 128, NB>(a, cache, grid, s);
    return launch<T, FORMAT, 256, NB>(a, cache, grid, s);
}

template <typename T, int FORMAT>
int launch_rows(Args& a, const TbB200Kv8* cache, dim3 grid, cudaStream_t s) {
    return a.block_rows == 8 ? launch_dim<T, FORMAT, 1>(a, cache, grid, s)
                             : launch_dim<T, FORMAT, 2>(a, cache, grid, s);
}

template <typename T, int W>
int join_by(const Args& a, int ctas, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas - 1, (unsigned)(a.block_rows * W * 32 / kJoinThreads));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_join<T, W>, a));
    TB_LAUNCH_CHECK("8-bit cache attention join kernel");
    return TB_OK;
}

// Four warps a row when few blocks have many parts each.
template <typename T>
int join(const Args& a, int ctas, cudaStream_t s) {
    return ctas > kManyParts * (int64_t)a.hkv * a.b.n_seqs ? join_by<T, 4>(a, ctas, s)
                                                          : join_by<T, 1>(a, ctas, s);
}

}  // namespace

extern "C" int tb_b200_kv8_attention_workspace(const TbB200Kv8* cache,
                                               const TbB200Kv8Batch* batch,
                                               const TbB200Kv8Attention* attention,
                                               size_t* bytes) {
    const int rc = check(cache, batch, attention, false);
    if (rc != TB_OK) return rc;
    if (!bytes) return TB_ERR_INVALID_ARG;
    *bytes = 0;
    if (batch->rows == 0 || batch->n_seqs == 0) return TB_OK;
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    if (kv8::chunk_suits(cache, batch, attention, ds->sm_count)) return TB_OK;
    *bytes = plan_of(cache, batch, attention, ds->sm_count).bytes();
    return TB_OK;
}

extern "C" int tb_b200_kv8_attention(const TbB200Kv8* cache, const TbB200Kv8Batch* batch,
                                     const TbB200Kv8Attention* attention, void* stream) {
    const TbB200Kv8Attention* t = attention;
    int rc = check(cache, batch, t, true);
    if (rc != TB_OK) return rc;
    if (batch->rows == 0 || batch->n_seqs == 0) return TB_OK;
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    if (kv8::chunk_suits(cache, batch, t, ds->sm_count))
        return kv8::chunk_attention(cache, batch, t, tbh::stream_of(stream));
    const Plan p = plan_of(cache, batch, t, ds->sm_count);
    const size_t bytes = p.bytes();
    if (bytes && (!t->workspace || t->workspace_bytes < bytes || !tbh::aligned16(t->workspace))) {
        tbh::set_error_text("8-bit cache attention: workspace missing, small or misaligned");
        return TB_ERR_INVALID_ARG;
    }
    const size_t s = t->dtype == TB_DTYPE_F32 ? 4 : 2;
    Args a = {};
    a.b = kv8::view(cache, batch);
    a.q = t->q;
    a.out = t->out;
    a.lse = t->lse;
    a.q_stride = t->q_stride;
    a.out_stride = t->out_stride;
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.status = ds->status;
    if (bytes) {
        uint8_t* w = static_cast<uint8_t*>(t->workspace);
        a.part = reinterpret_cast<float*>(w);
        a.state = reinterpret_cast<float2*>(w + p.part_bytes);
        a.cuts = reinterpret_cast<Cut*>(w + p.part_bytes + p.state_bytes);
    }
    a.scale = t->scale;
    a.hq = t->n_heads;
    a.hkv = cache->n_kv_heads;
    a.d = cache->head_dim;
    a.window = t->window;
    a.max_rows = t->max_rows;
    a.max_len = t->max_len;
    a.block_rows = p.block_rows;
    a.whole = p.whole;
    a.vec = tbh::aligned16(t->q) && t->q_stride * s % 16 == 0;
    a.vec_out = tbh::aligned16(t->out) && t->out_stride * s % 16 == 0;
    const dim3 grid((unsigned)p.ctas);
    cudaStream_t st = tbh::stream_of(stream);
    const bool f32 = t->dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    rc = f32 ? (int8 ? launch_rows<float, kv8::kInt8>(a, cache, grid, st)
                     : launch_rows<float, kv8::kE4m3>(a, cache, grid, st))
             : (int8 ? launch_rows<__nv_bfloat16, kv8::kInt8>(a, cache, grid, st)
                     : launch_rows<__nv_bfloat16, kv8::kE4m3>(a, cache, grid, st));
    if (rc != TB_OK || p.whole) return rc;
    return f32 ? join<float>(a, p.ctas, st) : join<__nv_bfloat16>(a, p.ctas, st);
}
