// k_mx_linear.cu -- y = x w^T (+ bias) of microscaled x [rows, cols] and w [outs, cols], on
// the block-scaled matrix instructions.
//
// w is the left operand: a tile is 128 outs by some rows of x, its sums in tensor memory as
// [out][row].  So a single row of x is as good a tile as many (the instruction takes 16 columns
// at least), and w, the larger side in serving, is read once for up to 256 rows.  Two shapes:
//
// Above 128 rows of x, two CTAs (a pair of SMs) have a tile of 256 outs by 256 rows together:
// each loads half of either operand, and the first one's products read both halves.  Codes and
// scales come by tensor copies of both CTAs that count on the first one's barriers: an arrival of
// the other CTA's own would release its shared memory first, 1500 clocks a step.  The scales of 128
// rows and 128 columns are 512 bytes that one copy of the tensor pipe brings from shared to tensor
// memory; two warps share those of a step.  A step of 256 columns (512 of 4 bits) takes 1170
// clocks, 1024 of them its products at the instruction's nominal rate; then it is the power limit
// that bounds long calls, by the clock.
//   4096 x 8192 x 28672, a few calls from a graph: 8-bit rows and 4-bit weights 632 us (3.0
//   PFLOP/s), both 8 bits 680, both 4 bits 325 (5.9 PFLOP/s); one after another for seconds 740 and
//   380 us (1432 MHz at 990 W); bf16 products of that size take 1150 us at the fastest.
//   Stores of scales from registers waited for the products in flight (4 bits: 806 us), copies by
//   one warp that asked for them too took 543, the other CTA's arrivals 420.  Steps of half the
//   columns, twice the stages: 1318 us for 632's case with those arrivals, 835 then.
//
// Up to 128 rows it is w's bytes that count, and the issuing warp's chain of waits, products and
// commits (1000 clocks a step of 128 columns): one tile of 128 outs a CTA, two CTAs an SM, one's
// loads under the other's epilogue, scales through registers (products are few, nothing waits for
// them).  Where the tiles leave SMs idle, the CTAs of a cluster take parts of cols and add them
// up, in order, through one another's shared memory; so do two of them in a last round that has
// tiles for half of the CTAs.
//   64 x 8192 x 128256, 4-bit weights to f32: 128 us (4.6 TB/s of the bytes there have to be);
//   one CTA an SM 419 us, three 152 against 135 then; last round whole 135 -> 130.
//   1 x 8192 x 57344: 57 us (4.4 TB/s); 64 with waits for a step that is there already.
//   1 x 4096 x 4096: 8.7 us, of which a launch and the first loads are the most.
//   Asking for w ahead into L2 made it slower (72 -> 85 us for 57344 outs), as did parts of cols
//   in every round.
#include <algorithm>
#include <atomic>

#include "mx.cuh"
#include "phases.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace {

// warps
constexpr int kLoader = 0, kIssuer = 1;
constexpr int kOuts = 128;  // of a CTA's tile
constexpr int kMostStages = 5, kMostAhead = 8, kMostSplit = 8;
constexpr int kPieceBytes = 128;  // of a row of codes; a step has one or two such pieces
constexpr uint64_t kLimit = 1000000000ull;  // ns, of a wait

struct Args {
    CUtensorMap w_map, x_map;
    CUtensorMap w_scale_map, x_scale_map;  // a pair's
    const uint8_t *w_scales, *x_scales;
    const float* bias;
    void* y;
    int64_t y_stride;
    unsigned* status;
    int rows, outs, tiles128;  // cols in tiles of 128
    int tile_rows, row_tiles, n_tiles;
    int steps, stages, stage_bytes, x_off, x_piece;
    int split, whole;  // CTAs that share a tile's steps; each one's tiles before, if split > 1
    int y_vec;       // rows of y start on 16 bytes
    int flat;        // a copy takes one piece, by its x
    int code_bytes;  // that a step's copies count, fill left out
    uint32_t columns, scales_column, instruction;
};

struct Shared {
    uint64_t full[kMostStages], scaled[kMostStages], empty[kMostStages];
    uint64_t asked[kMostAhead];  // a step's scales, to shared memory
    uint64_t sums, drained, products_done, scales_done;
    uint32_t tmem;
    int consumed, taken;  // steps whose codes, and whose scales, have been waited for
};

// A bounded wait.  The clock is read once in kTries tries (%globaltimer takes about a
// microsecond, as long as a step's products).
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, unsigned* status) {
    constexpr int kTries = 256;
    uint64_t t0 = 0;
    for (;;) {
        for (int i = 0; i < kTries; ++i)
            if (tbk::mbar_try_wait(bar, parity)) return true;
        const uint64_t now = tbk::global_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 > kLimit) break;
    }
    atomicOr(status, tbk::kFlagTimeout);
    return false;
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, unsigned* status) {
    const bool came = wait_one(bar, parity, status);
    return __all_sync(tbk::kFull, came);
}

// Whether a wait would be over.
__device__ __forceinline__ bool is_over(uint64_t* bar, uint32_t parity) {
    uint32_t over;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(over)
        : "r"(tbk::smem_addr(bar)), "r"(parity)
        : "memory");
    return over;
}

// `mine` in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer(const void* mine, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(at)
                 : "r"(tbk::smem_addr(mine)), "r"(rank));
    return at;
}
// Arrive on the first CTA's barrier, in the order of the tensor memory's accesses (tc::
// fence_before and its wait), which is all that it tells: with a release, of other memory too, it
// took some 1500 clocks.
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer(bar, 0))
                 : "memory");
}
// A tile to this CTA's shared memory; PAIR: counted on the first CTA's barrier.
template <bool PAIR>
__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, int x, int row,
                                         int piece, uint64_t* bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile"
            ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                tbk::smem_addr(dst)),
            "l"(map), "r"(x), "r"(row), "r"(piece), "r"(peer(bar, 0))
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tbk::smem_addr(dst)),
            "l"(map), "r"(x), "r"(row), "r"(piece), "r"(tbk::smem_addr(bar))
            : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float load_of(const float* mine, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(mine, rank)) : "memory");
    return v;
}

// A tile of n rows from `row` on and of outs from `out` on: the CTA's 128, or the pair's 256.
struct Tile {
    int out, row, n;
};
template <bool PAIR>
__device__ __forceinline__ Tile tile_of(const Args& a, int i) {
    constexpr int kUnit = PAIR ? 32 : 16;  // the instruction's, half of it in each CTA
    Tile t;
    t.out = i / a.row_tiles * (PAIR ? 2 * kOuts : kOuts);
    t.row = i % a.row_tiles * a.tile_rows;
    t.n = min(a.tile_rows, (a.rows - t.row + kUnit - 1) / kUnit * kUnit);
    return t;
}

// Steps [first, last) of a tile.
struct Work {
    Tile t;
    int first, last;
};

template <typename T, int N>
__device__ __forceinline__ void store_column(T* y, int64_t stride, int n, const float (&v)[N],
                                             float bias) {
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < n) tbk::Elt<T>::store(y + e * stride, v[e] + bias);
}

// PAIR: two CTAs on a tile of 256 outs by up to 256 rows, one an SM; else up to 128 rows.
template <bool BOTH4, bool PAIR>
struct Shape {
    static constexpr int kPieces = PAIR ? 2 : 1;
    static constexpr int kStoreWarps = PAIR ? 8 : 4;
    // warps: those that bring scales, and those that store
    static constexpr int kScalers = 2, kScaleWarps = PAIR ? 2 : 4, kStorers = 2 + kScaleWarps;
    static constexpr int kThreads = 32 * (kStorers + kStoreWarps);
    static constexpr int kTiles = (BOTH4 ? 2 : 1) * kPieces;  // of 128 columns, a step
    static constexpr int kMostX = PAIR ? 2 : 1;               // x's tiles of 128 rows
    static constexpr int kEach = (1 + kMostX) * kTiles;       // a step's tiles of scales
    static constexpr int kScaleColumns = 4 * kEach;
    static constexpr int kAhead = PAIR && BOTH4 ? 4 : 8;  // steps' scales asked for
    static constexpr int kScaleBytes = kAhead * kEach * mx::kTileBytes;
    static constexpr int kStaged = PAIR ? 8192 : 0;  // bytes of y on their way
};

// BOTH4: both operands 4-bit, a piece 256 columns; else 128.
template <typename T, bool BOTH4, bool PAIR>
__global__ void __launch_bounds__(Shape<BOTH4, PAIR>::kThreads, PAIR ? 1 : 2)
k_linear(const __grid_constant__ Args a) {
    using H = Shape<BOTH4, PAIR>;
    constexpr int kTiles = H::kTiles, kMostX = H::kMostX, kEach = H::kEach, kPieces = H::kPieces;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared sh;
    uint8_t* smem = smem_raw + (-tbk::smem_addr(smem_raw) & 1023u);
    // (the same in all lanes, and known to be)
    const int warp = __shfl_sync(tbk::kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int ctas = PAIR ? 2 : a.split, rank = blockIdx.x % ctas;
    // whole tiles, then, split > 1, a part of one that the cluster shares
    const int tile0 = PAIR ? blockIdx.x / 2 : blockIdx.x, tile_step = PAIR ? gridDim.x / 2 : gridDim.x;
    const int shared = a.whole * gridDim.x + blockIdx.x / ctas;
    const bool shares = !PAIR && a.split > 1 && shared < a.n_tiles;
    const int part_first = (int)((int64_t)a.steps * rank / ctas);
    const int part_last = (int)((int64_t)a.steps * (rank + 1) / ctas);
    const int whole = PAIR || a.split == 1 ? (a.n_tiles - 1 - tile0) / tile_step + 1 : a.whole;
    const int mine = whole + shares;
    const int total = whole * a.steps + (shares ? part_last - part_first : 0);  // this CTA's steps
    auto work_of = [&](int i) {
        Work w;
        const bool part = !PAIR && i == whole;
        w.t = tile_of<PAIR>(a, part ? shared : tile0 + i * tile_step);
        w.first = part ? part_first : 0;
        w.last = part ? part_last : a.steps;
        return w;
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            tbk::mbar_init(&sh.full[i], 1);
            tbk::mbar_init(&sh.scaled[i], H::kScaleWarps);
            tbk::mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < H::kAhead; ++i) tbk::mbar_init(&sh.asked[i], 1);
        tbk::mbar_init(&sh.scales_done, H::kScaleWarps);
        tbk::mbar_init(&sh.sums, 1);
        tbk::mbar_init(&sh.drained, (PAIR ? 2 : 1) * H::kStoreWarps);
        tbk::mbar_init(&sh.products_done, 1);
        sh.consumed = sh.taken = 0;
        tbk::fence_mbar_init();
    }
    if (warp == kIssuer) {
        if constexpr (PAIR)
            tc::allocate_pair(&sh.tmem, a.columns);
        else
            tc::allocate(&sh.tmem, a.columns);
    }
    tc::fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the other CTA's barriers are there
    tc::fence_after();
    const uint32_t tmem = sh.tmem;

    auto commit = [&](uint64_t* bar, bool leader) {
        if constexpr (PAIR)
            tc::commit_pair(bar, leader);
        else
            tc::commit(bar, leader);
    };
    int issued = 0, asked = 0;  // the loader's steps of codes and of scales
    bool fine = true;
    if (warp == kLoader) {
        if (lane == 0) {
            // PAIR: a step's scales too, to a ring of their own, kAhead steps before they are
            // taken
            constexpr int kAhead = H::kAhead;
            uint8_t* ring = smem + a.stages * a.stage_bytes;
            int ask_tile = 0, ask_step = 0, ask_slot = 0;  // the next that are asked for
            Tile ask_t = tile_of<PAIR>(a, tile0);
            auto ask = [&] {
                uint8_t* to = ring + ask_slot * kEach * mx::kTileBytes;
                uint64_t* bar = &sh.asked[ask_slot];
                const int at = ask_step * 2 * kTiles;  // (halves of a tile's scales)
                if (rank == 0) tbk::mbar_expect_tx(bar, 2 * kEach * mx::kTileBytes);
                tma_tile<PAIR>(to, &a.w_scale_map, 0, at, ask_t.out / kOuts + rank, bar);
                tma_tile<PAIR>(to + kTiles * mx::kTileBytes, &a.x_scale_map, 0, at,
                               ask_t.row / 128, bar);
                ++asked;
                if (++ask_slot == kAhead) ask_slot = 0;
                if (++ask_step == a.steps) {
                    ask_step = 0;
                    if (++ask_tile < mine) ask_t = tile_of<PAIR>(a, tile0 + ask_tile * tile_step);
                }
            };
            int stage = 0;
            uint32_t parity = 1;  // of the round before
            for (int i = 0; i < mine && fine; ++i) {
                const Work k = work_of(i);
                const int out = k.t.out + (PAIR ? kOuts * rank : 0);
                const int row = k.t.row + (PAIR ? k.t.n / 2 * rank : 0);
                for (int j = k.first; j < k.last; ++j) {
                    // the products of step issued - stages are done, and so are the copies of
                    // its scales
                    if (issued >= a.stages) fine = wait_one(&sh.empty[stage], parity, a.status);
                    if (!fine) break;
                    uint8_t* to = smem + stage * a.stage_bytes;
                    uint64_t* bar = &sh.full[stage];
                    if (!PAIR || rank == 0)
                        tbk::mbar_expect_tx(bar, (PAIR ? 2 : 1) * a.code_bytes);
                    if (PAIR && !a.flat) {
                        tma_tile<PAIR>(to, &a.w_map, 0, out, j * kPieces, bar);
                        tma_tile<PAIR>(to + a.x_off, &a.x_map, 0, row, j * kPieces, bar);
                    } else {
#pragma unroll
                        for (int p = 0; p < kPieces; ++p) {
                            const int x = (j * kPieces + p) * 128;  // (bytes, or 4-bit elements)
                            tma_tile<PAIR>(to + p * kOuts * kPieceBytes, &a.w_map, x, out, 0, bar);
                            tma_tile<PAIR>(to + a.x_off + p * a.x_piece, &a.x_map, x, row, 0, bar);
                        }
                    }
                    if constexpr (PAIR) {
                        while (asked < total && asked < kAhead + max(0, issued - a.stages + 1)) ask();
                    }
                    ++issued;
                    if (++stage == a.stages) {
                        stage = 0;
                        parity ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == kIssuer) {
        // A whole warp, one lane of which issues: operands stay in uniform registers (by one
        // lane's branch a step took twice the time).
        if (!PAIR || rank == 0) {
            const bool leader = lane == 0;
            const uint64_t w_desc = tc::tile_descriptor(tbk::smem_addr(smem), 16);
            const uint32_t x_off = a.x_off / 16, x_piece = a.x_piece / 16;
            int stage = 0, done = 0, consumed = 0;
            uint32_t parity = 0;
            // whether a step's operands are there is asked before the products of the step
            // before are issued: a wait that is over takes 220 clocks, a step's issue 340 to 600
            bool there = false;
            for (int i = 0; i < mine && fine; ++i) {
                const Work k = work_of(i);
                const uint32_t instruction = tc::with_columns(a.instruction, k.t.n);
                if (i > 0) fine = wait_all(&sh.drained, (i - 1) & 1, a.status);
                tc::fence_after();
                for (int j = k.first; j < k.last && fine; ++j) {
                    if (!there) fine = wait_all(&sh.full[stage], parity, a.status);
                    if (fine) ++consumed;
                    if (!there) fine = fine && wait_all(&sh.scaled[stage], parity, a.status);
                    if (!fine) break;
                    tc::fence_after();
                    const int next = stage + 1 == a.stages ? 0 : stage + 1;
                    const uint32_t next_parity = next ? parity : parity ^ 1;
                    const bool full = is_over(&sh.full[next], next_parity),
                               scaled = is_over(&sh.scaled[next], next_parity);
                    const uint32_t w_scales = tmem + a.scales_column + stage * H::kScaleColumns;
                    const uint32_t x_scales = w_scales + 4 * kTiles;
                    const uint64_t w = w_desc + (uint32_t)(stage * (a.stage_bytes / 16));
                    const int have = a.tiles128 - j * kTiles;  // the last step may have less
#pragma unroll
                    for (int p = 0; p < kPieces; ++p)
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const int h = BOTH4 ? 2 * p + m / 2 : p, block = BOTH4 ? m % 2 * 2 : m;
                            if (h == 0 || h < have)
                                tc::mma_scaled<BOTH4, PAIR>(
                                    tmem, w + p * (kOuts * kPieceBytes / 16) + 2 * m,
                                    w + x_off + p * x_piece + 2 * m,
                                    tc::with_block(instruction, block), w_scales + 4 * h,
                                    x_scales + 4 * kMostX * h, j > k.first || p + m > 0, leader);
                        }
                    if (done + a.stages < total) commit(&sh.empty[stage], leader);
                    ++done;
                    stage = next;
                    parity = next_parity;
                    there = __all_sync(tbk::kFull, full && scaled);
                }
                if (fine) commit(&sh.sums, leader);
            }
            if (leader) sh.consumed = consumed;
            // whatever ended the loop, no product may be in flight when tensor memory is freed
            commit(&sh.products_done, leader);
            wait_all(&sh.products_done, 0, a.status);
        }
    } else if (warp < H::kStorers) {
        if constexpr (PAIR) {
            // Two warps, half of a step's copies of scales to tensor memory each.
            constexpr int kAhead = H::kAhead;
            const int part = warp - H::kScalers;
            const bool leader = lane == 0;
            const uint8_t* ring = smem + a.stages * a.stage_bytes;
            int stage = 0, slot = 0, step = 0;
            uint32_t parity = 0, slot_parity = 0;
            for (int done = 0; done < total && rank == 0; ++done) {
                fine = wait_all(&sh.asked[slot], slot_parity, a.status);
                if (!fine) break;
                if (part == 0 && lane == 0) sh.taken = done + 1;
                if (done >= a.stages) fine = wait_all(&sh.empty[stage], parity ^ 1, a.status);
                if (!fine) break;
                tc::fence_after();
                const uint32_t from = tbk::smem_addr(ring) + slot * kEach * mx::kTileBytes;
                const uint32_t w_to = tmem + a.scales_column + stage * H::kScaleColumns;
                const uint32_t x_to = w_to + 4 * kTiles;
                const int have = a.tiles128 - step * kTiles;
#pragma unroll
                for (int i = 0; i < kTiles / 2; ++i) {
                    const int h = 2 * i + part;
                    if (h >= have) break;
                    tc::copy_scales(w_to + 4 * h, from + h * mx::kTileBytes, leader);
#pragma unroll
                    for (int k = 0; k < kMostX; ++k)
                        tc::copy_scales(x_to + 4 * (kMostX * h + k),
                                        from + ((1 + k) * kTiles + h) * mx::kTileBytes, leader);
                }
                // (by the first CTA alone: the other's issuer does not wait)
                tc::commit_of_pair(&sh.scaled[stage], leader);
                if (++step == a.steps) step = 0;
                if (++slot == kAhead) {
                    slot = 0;
                    slot_parity ^= 1;
                }
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            if (rank == 0) {
                // no copy to tensor memory may be in flight when that is freed
                tc::commit_of_pair(&sh.scales_done, leader);
                wait_all(&sh.scales_done, 0, a.status);
            }
        } else {
            // Four warps: scales to shared memory, kAhead - 1 steps ahead, by all of them; from
            // there through registers, each to its quarter of the rows of tensor memory, a lane
            // the words of rows l, l + 32, l + 64 and l + 96.
            constexpr int kAhead = H::kAhead, kChunks = kEach * 32;
            const uint32_t to = tmem + a.scales_column + ((uint32_t)(warp % 4) << 21);
            const int thread = threadIdx.x - 32 * H::kScalers;
            uint4* ring = reinterpret_cast<uint4*>(smem + a.stages * a.stage_bytes);
            int ask_tile = 0, ask_slot = 0;
            Work next = work_of(0);  // the next step that is asked for is its first
            auto ask = [&] {
                if (ask_tile < mine) {
                    const Tile t = next.t;
#pragma unroll
                    for (int i = 0; i < (kChunks + 127) / 128; ++i) {
                        const int c = thread + 128 * i, tile = c / 32, x = tile - kTiles;
                        const int h = x < 0 ? tile : x / kMostX, at = next.first * kTiles + h;
                        const int row = x < 0 ? t.out : t.row + 128 * (x % kMostX);
                        if (c < kChunks && at < a.tiles128 && row < (x < 0 ? a.outs : a.rows)) {
                            const uint8_t* from = (x < 0 ? a.w_scales : a.x_scales) +
                                                  mx::scales_at(row, at, a.tiles128) + c % 32 * 16;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                             tbk::smem_addr(ring + ask_slot * kChunks + c)),
                                         "l"(from)
                                         : "memory");
                        }
                    }
                    if (++next.first == next.last && ++ask_tile < mine) next = work_of(ask_tile);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++ask_slot == kAhead) ask_slot = 0;
            };
#pragma unroll 1
            for (int i = 0; i < kAhead - 1; ++i) ask();
            int stage = 0, slot = 0;
            uint32_t parity = 1;  // of the round before
            for (int done = 0; done < total; ++done) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
                // this step's are there, and the step before's have been taken by all
                asm volatile("bar.sync 1, 128;" ::: "memory");
                ask();
                uint4 r[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) r[i] = ring[slot * kChunks + i * 32 + lane];
                if (done >= a.stages) {
                    if (fine) fine = wait_all(&sh.empty[stage], parity, a.status);
                }
                if (fine) {  // (a warp that gave up still comes to the barrier above)
                    tc::fence_after();
                    const uint32_t at = to + stage * H::kScaleColumns;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) tc::store_scales(at + 4 * i, r[i]);
                    tc::wait_store();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tbk::mbar_arrive(&sh.scaled[stage]);
                }
                if (++slot == kAhead) slot = 0;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        const int quarter = warp % 4;
        const uint32_t sums = tmem + ((uint32_t)quarter << 21);
        float* part = reinterpret_cast<float*>(smem);  // of a shared tile: [row][out]
        for (int i = 0; i < mine; ++i) {
            const Tile t = work_of(i).t;
            if (fine) fine = wait_all(&sh.sums, i & 1, a.status);
            if (!fine && !PAIR) break;  // (a pair's warps still come to the barriers below)
            tc::fence_after();
            const int out = t.out + (PAIR ? kOuts * rank : 0) + 32 * quarter + lane;
            const float bias = a.bias && out < a.outs ? a.bias[out] : 0.0f;
            const int n = out < a.outs ? min(a.rows - t.row, t.n) : 0;
            T* y = static_cast<T*>(a.y) + (int64_t)t.row * a.y_stride + out;
            auto release = [&] {  // tensor memory may take the next tile's sums
                tc::fence_before();
                __syncwarp();
                if (lane == 0 && i + 1 < mine) {
                    if (PAIR)
                        arrive_first(&sh.drained);
                    else
                        tbk::mbar_arrive(&sh.drained);
                }
            };
            if constexpr (PAIR) {
                // half of the rows each of two warps, in registers before any is stored; then
                // through shared memory, for whole rows of the CTA's outs to be stored at once
                constexpr int kRows = H::kStaged / 2 / (kOuts * sizeof(T));  // of each half
                constexpr int kVec = 16 / sizeof(T), kPer = kOuts / kVec;    // pieces of a row
                const int half = (warp - H::kStorers) / 4, c = half * 128;
                const int thread = threadIdx.x - 32 * H::kStorers;
                T* staged = reinterpret_cast<T*>(smem + a.stages * a.stage_bytes + H::kScaleBytes);
                T* y0 = static_cast<T*>(a.y) + (int64_t)t.row * a.y_stride + t.out + kOuts * rank;
                const int outs = a.outs - t.out - kOuts * rank, rows = min(a.rows - t.row, t.n);
                float v[128];
                if (c < t.n) tc::load<128>(sums + c, v);
                if (fine) release();
#pragma unroll
                for (int g = 0; g < 128; g += kRows) {
                    if (g >= t.n) break;
#pragma unroll
                    for (int e = 0; e < kRows; ++e)
                        tbk::Elt<T>::store(staged + (half * kRows + e) * kOuts + 32 * quarter + lane,
                                           v[g + e] + bias);
                    asm volatile("bar.sync 2, 256;" ::: "memory");
#pragma unroll
                    for (int k = 0; k < 2 * kRows * kPer / 256; ++k) {
                        const int i = thread + 256 * k, r = i / kPer, o = i % kPer * kVec;
                        const int row = r / kRows * 128 + g + r % kRows;
                        if (row >= rows || o >= outs) continue;
                        const T* from = staged + r * kOuts + o;
                        T* to = y0 + (int64_t)row * a.y_stride + o;
                        if (a.y_vec && o + kVec <= outs) {
                            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
                        } else {
                            for (int e = 0; e < kVec && o + e < outs; ++e) to[e] = from[e];
                        }
                    }
                    asm volatile("bar.sync 2, 256;" ::: "memory");
                }
            } else {
                for (int c = 0; c < t.n; c += 32) {
                    float v[32];
                    tc::load<32>(sums + c, v);
                    if (i == whole) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (c + e < t.n) part[(c + e) * kOuts + 32 * quarter + lane] = v[e];
                    } else {
                        store_column(y + c * a.y_stride, a.y_stride, n - c, v, bias);
                    }
                }
                release();
            }
        }
    }
    tc::fence_before();
    const bool lost = __syncthreads_or(!fine);
    if (warp == kLoader && lane == 0 && lost && (!PAIR || rank == 0)) {
        // no copy may be in flight when the CTA ends: those that nobody waited for (a pair's
        // other CTA is behind the barrier below until then)
        for (int j = sh.consumed; j < issued; ++j)
            wait_one(&sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u, a.status);
    }
    if (PAIR && rank == 0 && warp == kLoader && lane == 0 && lost) {
        for (int j = sh.taken; j < asked; ++j)
            wait_one(&sh.asked[j % H::kAhead], (uint32_t)(j / H::kAhead) & 1u, a.status);
    }
    __syncwarp();
    if constexpr (PAIR) {
        // (the first CTA's last arrival comes here too)
        if (warp == kIssuer && rank == 1) wait_all(&sh.products_done, 0, a.status);
        cluster_sync();  // no product reads the other's shared memory any more
        if (warp == kIssuer) tc::release_pair(tmem, a.columns);
        return;
    }
    if (warp == kIssuer) tc::release(tmem, a.columns);
    if (shares) {
        cluster_sync();
        if (warp >= H::kStorers) {
            const Tile t = tile_of<PAIR>(a, shared);
            const int at = warp % 4 * 32 + lane, out = t.out + at;
            if (out < a.outs) {
                const float bias = a.bias ? a.bias[out] : 0.0f;
                const int n = min(a.rows - t.row, t.n);
                const float* part = reinterpret_cast<const float*>(smem) + at;
                for (int c = rank; c < n; c += a.split) {
                    float sum = 0.0f;
                    for (int k = 0; k < a.split; ++k) sum += load_of(part + c * kOuts, k);
                    tbk::Elt<T>::store(static_cast<T*>(a.y) + (t.row + c) * a.y_stride + out,
                                       sum + bias);
                }
            }
        }
        cluster_sync();  // the others have read this CTA's part
    }
}

struct Plan {
    bool pair;
    int tile_rows, row_tiles, n_tiles, steps, split, whole, stages, stage_bytes, bytes, ctas;
    int x_rows;  // that a CTA loads
    uint32_t columns, scales_column;
};

int plan_of(Plan& p, const TbB200Mx* x, const TbB200Mx* w, bool both4, int sm_count) {
    const int64_t tiles128 = mx::tiles_of(x->cols);
    // In us, single CTAs and pairs at 64, 96, 128, 129 and 256 rows (above 128 single ones read w
    // again for each 128), 8-bit rows and 4-bit weights:
    //   8192 x 8192    18 24   21 24   24 25   37 26   38 28
    //   8192 x 28672   34 43   40 44   43 46   72 47   75 55
    //   8192 x 57344   66 81   78 83   82 86  144 89  147 106
    //   28672 x 8192   38 67   44 68   47 71   76 73   78 82
    //   4096 x 4096    13 13   15 14   17 14   19 15   20 16
    //   4096 x 11008   20 15   25 15   29 15   24 16   24 18
    //   8192 x 28672, both 4 bits  29 30, 36 32 at 128, 55 32, 59 35
    // 128 is where pairs take over for the larger of these; of short cols they are ahead from 32
    // to 96 rows on, which the rule leaves.
    p.pair = x->rows > 128;
    const int pieces = p.pair ? 2 : 1, step_tiles = (both4 ? 2 : 1) * pieces;
    p.steps = (int)((tiles128 + step_tiles - 1) / step_tiles);
    p.tile_rows = p.pair ? 256 : (int)((x->rows + 15) / 16 * 16);
    p.x_rows = p.pair ? 128 : p.tile_rows;
    p.row_tiles = (int)((x->rows + p.tile_rows - 1) / p.tile_rows);
    const int outs = p.pair ? 2 * kOuts : kOuts;
    const int64_t n_tiles = (w->rows + outs - 1) / outs * p.row_tiles;
    if (n_tiles * kMostSplit > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    p.n_tiles = (int)n_tiles;
    p.stage_bytes = pieces * (kOuts + p.x_rows) * kPieceBytes;
    const int scales = p.pair ? Shape<false, true>::kScaleBytes
                       : both4 ? Shape<true, false>::kScaleBytes : Shape<false, false>::kScaleBytes;
    static_assert(Shape<false, true>::kScaleBytes == Shape<true, true>::kScaleBytes, "scales");
    const int beside = scales + (p.pair ? Shape<false, true>::kStaged : 0) + 1024;
    const int per_sm = p.pair ? 1 : 2;
    p.stages = (226 * 1024 / per_sm - 1024 - beside) / p.stage_bytes;
    static_assert((226 * 1024 / 2 - 2048 - Shape<false, false>::kScaleBytes) /
                          ((kOuts + 16) * kPieceBytes) <= kMostStages, "the smallest tiles' stages");
    p.scales_column = (uint32_t)(p.tile_rows + 31) / 32 * 32;
    const int scale_columns = (p.pair ? 12 : 8) * step_tiles;
    const uint32_t need = p.scales_column + p.stages * scale_columns;
    for (p.columns = 32; p.columns < need;) p.columns *= 2;
    const int slots = p.pair ? sm_count / 2 : sm_count * per_sm;
    // parts of cols, 4 steps each at least: where the tiles leave SMs idle, and of the last
    // round's tiles where they are for half of the CTAs or fewer
    const int rest = (int)(n_tiles % slots);
    const bool can = !p.pair && p.tile_rows * kOuts * 4 <= p.stages * p.stage_bytes;
    p.split = 1;
    p.whole = 0;
    if (n_tiles > slots) {
        if (can && rest && 2 * rest <= slots && p.steps >= 8) {
            p.split = 2;
            p.whole = (int)(n_tiles / slots);
        }
    } else if (can) {
        // clusters of 3, 5, 6 or 7 leave places of a GPC over, up to one less than their CTAs:
        // those of 3 that fit take 10.4 us for 11.9 (1 x 4096 x 11008), ones too many 25 for 18
        constexpr int kGpcs = 8;
        p.split = (int)std::min<int64_t>({kMostSplit, slots / n_tiles, std::max(p.steps / 4, 1)});
        while ((p.split & (p.split - 1)) && n_tiles * p.split > slots - kGpcs * (p.split - 1))
            --p.split;
    }
    p.ctas = n_tiles > slots ? slots : p.n_tiles * p.split;
    if (p.pair) p.ctas *= 2;
    p.bytes = p.stages * p.stage_bytes + beside;
    return TB_OK;
}

// Tiles of `rows` rows and one piece of 128 bytes, or (not flat) two pieces, one after the
// other in shared memory: codes packed, or with fill beside 8-bit codes.
int map_of(CUtensorMap* map, const TbB200Mx* t, int rows, bool flat, bool packed) {
    const uint64_t pitch = (uint64_t)mx::pitch_of(t->format, t->cols);
    const bool fill = t->format == mx::kE2m1 && !packed;
    const uint64_t wide = fill ? kPieceBytes / 2 : kPieceBytes;  // a piece's bytes in memory
    const uint64_t dims[3] = {flat ? pitch * kPieceBytes / wide : kPieceBytes, (uint64_t)t->rows,
                              flat ? 1 : pitch / wide};
    const uint64_t strides[2] = {pitch, flat ? pitch * (uint64_t)t->rows : wide};
    const uint32_t box[3] = {kPieceBytes, (uint32_t)rows, flat ? 1u : 2u};
    return fill ? tbh::encode_tiles_u4(map, t->codes, dims, strides, box, 128)
                : tbh::encode_tiles_u8(map, t->codes, dims, strides, box, 128);
}

// The scales of a step's `tiles` tiles of 128 columns and of 128 or 256 rows: whole boxes, with
// zeros where the tensor has ended.
int scale_map_of(CUtensorMap* map, const TbB200Mx* t, int tiles, int row_tiles) {
    const uint64_t n = (uint64_t)mx::tiles_of(t->cols);
    const uint64_t dims[3] = {mx::kTileBytes / 2, 2 * n, (uint64_t)mx::tiles_of(t->rows)};
    const uint64_t strides[2] = {mx::kTileBytes / 2, n * mx::kTileBytes};
    const uint32_t box[3] = {mx::kTileBytes / 2, 2u * tiles, (uint32_t)row_tiles};
    return tbh::encode_tiles_u8(map, t->scales, dims, strides, box, 0);
}

template <typename T, bool BOTH4, bool PAIR>
int launch(const Args& a, const Plan& p, cudaStream_t s) {
    static std::atomic<uint64_t> granted{0};  // a bit per device
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    if (!(granted.load() >> ds->device & 1)) {
        TB_CUDA_TRY(cudaFuncSetAttribute(k_linear<T, BOTH4, PAIR>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
        granted.fetch_or(1ull << ds->device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.ctas);
    cfg.blockDim = dim3(Shape<BOTH4, PAIR>::kThreads);
    cfg.dynamicSmemBytes = (size_t)p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(PAIR ? 2 : p.split);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_linear<T, BOTH4, PAIR>, a));
    TB_LAUNCH_CHECK("microscaled product kernel");
    return TB_OK;
}

template <typename T>
int launch_by(const Args& a, const Plan& p, bool both4, cudaStream_t s) {
    if (p.pair) return both4 ? launch<T, true, true>(a, p, s) : launch<T, false, true>(a, p, s);
    return both4 ? launch<T, true, false>(a, p, s) : launch<T, false, false>(a, p, s);
}

tc::Element element(int format) { return format == mx::kE4m3 ? tc::kE4m3 : tc::kE2m1; }

}  // namespace

extern "C" int tb_b200_mx_linear(const TbB200Mx* x, const TbB200Mx* w, const float* bias,
                                 int out_dtype, void* y, int64_t y_stride, void* stream) {
    int rc = mx::check(x, true);
    if (rc == TB_OK) rc = mx::check(w, true);
    if (rc != TB_OK) return rc;
    if (out_dtype != TB_DTYPE_F32 && out_dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (x->cols != w->cols || (x->rows > 1 && y_stride < w->rows)) return TB_ERR_INVALID_SHAPE;
    if (x->rows == 0 || w->rows == 0) return TB_OK;
    if (!y) return TB_ERR_INVALID_ARG;
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    const bool both4 = x->format == mx::kE2m1 && w->format == mx::kE2m1;
    Plan p = {};
    rc = plan_of(p, x, w, both4, ds->sm_count);
    if (rc != TB_OK) return rc;
    Args a = {};
    // (rows that end within a piece of packed codes are not whole pieces)
    const int pieces = p.pair ? 2 : 1;
    a.flat = !p.pair || (both4 && mx::tiles_of(x->cols) % 2);
    rc = map_of(&a.w_map, w, kOuts, a.flat, both4);
    if (rc == TB_OK) rc = map_of(&a.x_map, x, p.x_rows, a.flat, both4);
    if (p.pair) {
        const int tiles = both4 ? 4 : 2;
        if (rc == TB_OK) rc = scale_map_of(&a.w_scale_map, w, tiles, 1);
        if (rc == TB_OK) rc = scale_map_of(&a.x_scale_map, x, tiles, 2);
    }
    if (rc != TB_OK) return rc;
    a.w_scales = w->scales;
    a.x_scales = x->scales;
    a.bias = bias;
    a.y = y;
    a.y_stride = y_stride;
    a.y_vec = tbh::aligned16(y) && y_stride * (out_dtype == TB_DTYPE_F32 ? 4 : 2) % 16 == 0;
    a.status = ds->status;
    a.rows = (int)x->rows;
    a.outs = (int)w->rows;
    a.tiles128 = (int)mx::tiles_of(x->cols);
    a.tile_rows = p.tile_rows;
    a.row_tiles = p.row_tiles;
    a.n_tiles = p.n_tiles;
    a.steps = p.steps;
    a.split = p.split;
    a.whole = p.whole;
    a.stages = p.stages;
    a.stage_bytes = p.stage_bytes;
    a.x_off = pieces * kOuts * kPieceBytes;
    a.x_piece = p.x_rows * kPieceBytes;
    a.code_bytes = pieces * ((kOuts * kPieceBytes >> (w->format == mx::kE2m1 && !both4)) +
                              (p.x_rows * kPieceBytes >> (x->format == mx::kE2m1 && !both4)));
    a.columns = p.columns;
    a.scales_column = p.scales_column;
    const int m = p.pair ? 2 * kOuts : kOuts;
    a.instruction = both4 ? tc::scaled_instruction_4bit(m)
                          : tc::scaled_instruction(element(w->format), element(x->format), m);
    cudaStream_t s = tbh::stream_of(stream);
    return out_dtype == TB_DTYPE_F32 ? launch_by<float>(a, p, both4, s)
                                     : launch_by<__nv_bfloat16>(a, p, both4, s);
}
