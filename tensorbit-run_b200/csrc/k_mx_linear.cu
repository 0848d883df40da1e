// k_mx_linear.cu -- y = x w^T (+ bias) of microscaled x [rows, cols] and w [outs, cols], on
// the block-scaled matrix instructions.
//
// w is the left operand: a tile is 128 outs by up to 256 rows of x, its sums in tensor memory
// as [out][row].  So a single row of x is as good a tile as many (the instruction takes 16
// columns at least), and w, the larger side in serving, is read once for up to 256 rows.
// One warp asks for operands and scales by TMA, one copies the scales to tensor memory and
// issues the products, four bring a tile's sums to y, a lane an out.  Where the tiles do not
// fill the SMs, the CTAs of a cluster take parts of cols and add them up, in order, through
// one another's shared memory.
#include <atomic>

#include "mx.cuh"
#include "phases.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace {

constexpr int kThreads = 192;
constexpr int kLoader = 0, kIssuer = 1, kStoreWarps = 4;  // warps; the others store
constexpr int kTileOuts = 128, kMostRows = 256, kMostStages = 12, kMostSplit = 8;
constexpr int kStepBytes = 128;  // of a row of codes

struct Args {
    CUtensorMap w_map, x_map;
    const uint8_t *w_scales, *x_scales;
    const float* bias;
    void* y;
    int64_t y_stride;
    unsigned* status;
    int rows, outs, tiles128;  // cols in tiles of 128
    int tile_rows, row_tiles, n_tiles;
    int steps, split, stages, stage_bytes, scales_off;
    int code_bytes;  // that a step's copies of codes count, fill left out
    uint32_t columns, scales_column, instruction;
};

struct Shared {
    uint64_t full[kMostStages], empty[kMostStages], sums, drained, products_done;
    uint32_t tmem;
    int consumed;  // steps whose operands the issuer has waited for
};

__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, unsigned* status) {
    const bool came = tbk::mbar_wait(bar, parity, status, 1000000000ull);
    return __all_sync(tbk::kFull, came);
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, int x, int y,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tbk::smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(0), "r"(tbk::smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float load_of(uint32_t smem, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// A tile of rows [row, row + n) and outs [out, out + 128).
struct Tile {
    int out, row, n, scale_tiles;
};
__device__ __forceinline__ Tile tile_of(const Args& a, int i) {
    Tile t;
    t.out = i / a.row_tiles * kTileOuts;
    t.row = i % a.row_tiles * a.tile_rows;
    t.n = min(a.tile_rows, (a.rows - t.row + 15) / 16 * 16);
    t.scale_tiles = (t.n + 127) / 128;
    return t;
}

// BOTH4: both operands 4-bit, a step 256 columns; else 128.
template <typename T, bool BOTH4>
__global__ void __launch_bounds__(kThreads) k_linear(const __grid_constant__ Args a) {
    constexpr int kScaleTiles = BOTH4 ? 2 : 1;  // of 4 blocks, a step
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared sh;
    uint8_t* smem = smem_raw + (-tbk::smem_addr(smem_raw) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.split;
    const int first = (int)((int64_t)a.steps * rank / a.split);
    const int last = (int)((int64_t)a.steps * (rank + 1) / a.split);
    const int tile0 = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
    const int mine = tile0 < a.n_tiles ? (a.n_tiles - 1 - tile0) / tile_step + 1 : 0;
    const int total = mine * (last - first);  // steps of this CTA
    auto stage_at = [&](int stage) { return smem + stage * a.stage_bytes; };

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            tbk::mbar_init(&sh.full[i], 1);
            tbk::mbar_init(&sh.empty[i], 1);
        }
        tbk::mbar_init(&sh.sums, 1);
        tbk::mbar_init(&sh.drained, kStoreWarps);
        tbk::mbar_init(&sh.products_done, 1);
        tbk::fence_mbar_init();
    }
    if (warp == kIssuer) tc::allocate(&sh.tmem, a.columns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = sh.tmem;

    int issued = 0;
    bool fine = true;
    if (warp == kLoader) {
        int stage = 0;
        uint32_t parity = 1;  // of the round before
        for (int i = 0; i < mine && fine; ++i) {
            const Tile t = tile_of(a, tile0 + i * tile_step);
            for (int j = first; j < last; ++j) {
                if (issued >= a.stages) fine = wait_all(&sh.empty[stage], parity, a.status);
                if (!fine) break;
                if (lane == 0) {
                    uint8_t* to = stage_at(stage);
                    uint64_t* bar = &sh.full[stage];
                    // (the last step of 256 columns may have 128)
                    const int at = j * kScaleTiles;
                    const int bytes = min(kScaleTiles, a.tiles128 - at) * mx::kTileBytes;
                    tbk::mbar_expect_tx(bar, a.code_bytes + (1 + t.scale_tiles) * bytes);
                    tma_tile(to, &a.w_map, j * 128, t.out, bar);
                    tma_tile(to + kTileOuts * kStepBytes, &a.x_map, j * 128, t.row, bar);
                    uint8_t* s = to + a.scales_off;
                    tbk::bulk_g2s(s, a.w_scales + mx::scales_at(t.out, at, a.tiles128), bytes, bar);
                    for (int k = 0; k < t.scale_tiles; ++k)
                        tbk::bulk_g2s(s + (1 + k) * kScaleTiles * mx::kTileBytes,
                                      a.x_scales + mx::scales_at(t.row + 128 * k, at, a.tiles128),
                                      bytes, bar);
                }
                __syncwarp();
                ++issued;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp == kIssuer) {
        const bool leader = lane == 0;
        const uint64_t w_desc = tc::tile_descriptor(tbk::smem_addr(smem), 16);
        const uint64_t x_desc = w_desc + kTileOuts * kStepBytes / 16;
        const uint32_t scales_s = tbk::smem_addr(smem) + a.scales_off;
        const int scale_columns = (1 + (a.tile_rows + 127) / 128) * kScaleTiles * 4;
        int stage = 0, done = 0;
        uint32_t parity = 0;
        for (int i = 0; i < mine && fine; ++i) {
            const Tile t = tile_of(a, tile0 + i * tile_step);
            const uint32_t instruction = tc::with_columns(a.instruction, t.n);
            if (i > 0) fine = wait_all(&sh.drained, (i - 1) & 1, a.status);
            tc::fence_after();
            for (int j = first; j < last && fine; ++j) {
                fine = wait_all(&sh.full[stage], parity, a.status);
                if (!fine) break;
                const uint32_t s = scales_s + stage * a.stage_bytes;
                const uint32_t w_to = tmem + a.scales_column + stage * scale_columns;
                const uint32_t x_to = w_to + kScaleTiles * 4;
                const int have = min(kScaleTiles, a.tiles128 - j * kScaleTiles);
                for (int h = 0; h < have; ++h) {
                    tc::copy_scales(w_to + 4 * h, s + h * mx::kTileBytes, leader);
                    // rows' tiles one after the other for each 4 blocks
                    for (int k = 0; k < t.scale_tiles; ++k)
                        tc::copy_scales(x_to + (h * t.scale_tiles + k) * 4,
                                        s + ((1 + k) * kScaleTiles + h) * mx::kTileBytes, leader);
                }
                const uint64_t off = stage * (a.stage_bytes / 16);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int h = BOTH4 ? m / 2 : 0, block = BOTH4 ? m % 2 * 2 : m;
                    if (h < have)
                        tc::mma_scaled<BOTH4>(tmem, w_desc + off + 2 * m, x_desc + off + 2 * m,
                                              tc::with_block(instruction, block), w_to + 4 * h,
                                              x_to + h * t.scale_tiles * 4, j > first || m > 0,
                                              leader);
                }
                if (done + a.stages < total) tc::commit(&sh.empty[stage], leader);
                ++done;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            if (fine) tc::commit(&sh.sums, leader);
        }
        if (lane == 0) sh.consumed = done;
        // whatever ended the loop, no product may be in flight when tensor memory is freed
        tc::commit(&sh.products_done, leader);
        wait_all(&sh.products_done, 0, a.status);
    } else {
        const int quarter = warp % 4;
        const uint32_t sums = tmem + ((uint32_t)quarter << 21);
        float* part = reinterpret_cast<float*>(smem);  // split: [row][out]
        for (int i = 0; i < mine; ++i) {
            const Tile t = tile_of(a, tile0 + i * tile_step);
            fine = wait_all(&sh.sums, i & 1, a.status);
            if (!fine) break;
            tc::fence_after();
            const int out = t.out + 32 * quarter + lane;
            const float bias = a.bias && out < a.outs ? a.bias[out] : 0.0f;
            T* y = static_cast<T*>(a.y) + (int64_t)t.row * a.y_stride + out;
            for (int c = 0; c < t.n; c += 32) {
                float v[32];
                tc::load<32>(sums + c, v);
                if (a.split > 1) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (c + e < t.n) part[(c + e) * kTileOuts + 32 * quarter + lane] = v[e];
                } else if (out < a.outs) {
                    const int n = min(a.rows - t.row, t.n) - c;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (e < n) tbk::Elt<T>::store(y + (c + e) * a.y_stride, v[e] + bias);
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0 && i + 1 < mine) tbk::mbar_arrive(&sh.drained);
        }
    }
    tc::fence_before();
    const bool lost = __syncthreads_or(!fine);
    if (warp == kLoader && lost) {
        // no copy may be in flight when the CTA ends: those that nobody waited for
        for (int j = sh.consumed; j < issued; ++j)
            wait_all(&sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u, a.status);
    }
    if (warp == kIssuer) tc::release(tmem, a.columns);
    if (a.split > 1) {
        cluster_sync();
        if (warp >= 2) {
            const Tile t = tile_of(a, tile0);
            const int quarter = warp % 4, out = t.out + 32 * quarter + lane;
            if (out < a.outs) {
                const float bias = a.bias ? a.bias[out] : 0.0f;
                const int n = min(a.rows - t.row, t.n);
                for (int c = rank; c < n; c += a.split) {
                    const uint32_t at =
                        tbk::smem_addr(smem) + (c * kTileOuts + 32 * quarter + lane) * 4;
                    float sum = 0.0f;
                    for (int k = 0; k < a.split; ++k) sum += load_of(at, k);
                    tbk::Elt<T>::store(static_cast<T*>(a.y) + (t.row + c) * a.y_stride + out,
                                       sum + bias);
                }
            }
        }
        cluster_sync();  // the others have read this CTA's part
    }
}

struct Plan {
    int tile_rows, row_tiles, n_tiles, steps, split, stages, stage_bytes, scales_off, bytes, ctas;
    uint32_t columns, scales_column;
};

int plan_of(Plan& p, const TbB200Mx* x, const TbB200Mx* w, bool both4, int sm_count) {
    const int64_t tiles128 = mx::tiles_of(x->cols);
    p.tile_rows = x->rows >= kMostRows ? kMostRows : (int)((x->rows + 15) / 16 * 16);
    p.row_tiles = (int)((x->rows + p.tile_rows - 1) / p.tile_rows);
    const int64_t n_tiles = (w->rows + kTileOuts - 1) / kTileOuts * p.row_tiles;
    if (n_tiles * kMostSplit > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    p.n_tiles = (int)n_tiles;
    p.steps = (int)(both4 ? (tiles128 + 1) / 2 : tiles128);
    const int scale_tiles = (1 + (p.tile_rows + 127) / 128) * (both4 ? 2 : 1);
    p.scales_off = (kTileOuts + p.tile_rows) * kStepBytes;
    p.stage_bytes = p.scales_off + (scale_tiles * mx::kTileBytes + 1023) / 1024 * 1024;
    const int per_sm = p.tile_rows <= 64 ? 2 : 1;
    const int budget = (per_sm == 2 ? 112 : 224) * 1024;
    p.stages = (budget - 1024) / p.stage_bytes;
    if (p.stages > kMostStages) p.stages = kMostStages;
    p.scales_column = (uint32_t)(p.tile_rows + 31) / 32 * 32;
    const uint32_t need = p.scales_column + p.stages * scale_tiles * 4;
    for (p.columns = 32; p.columns < need;) p.columns *= 2;
    const int slots = sm_count * per_sm;
    // parts of cols: rounds of CTAs by what each takes, a tile's fixed cost as 8 steps
    p.split = 1;
    int64_t best = INT64_MAX;
    for (int s = 1; s <= kMostSplit; s *= 2) {
        if (s > 1 && (p.steps < 2 * s || p.tile_rows * kTileOuts * 4 > p.stages * p.stage_bytes))
            break;
        const int64_t rounds = (n_tiles * s + slots - 1) / slots;
        const int64_t cost = rounds * ((p.steps + s - 1) / s + 8);
        if (cost < best) {
            best = cost;
            p.split = s;
        }
    }
    p.ctas = p.split > 1 ? p.n_tiles * p.split : p.n_tiles < slots ? p.n_tiles : slots;
    p.bytes = p.stages * p.stage_bytes + 1024;
    return TB_OK;
}

// Rows of 128 bytes of codes a step: packed, or with fill beside 8-bit codes.
int map_of(CUtensorMap* map, const TbB200Mx* t, int rows, bool packed) {
    const uint64_t pitch = (uint64_t)mx::pitch_of(t->format, t->cols);
    const uint64_t strides[2] = {pitch, pitch * (uint64_t)t->rows};
    const uint32_t box[3] = {128, (uint32_t)rows, 1};
    if (t->format == mx::kE2m1 && !packed) {
        const uint64_t dims[3] = {2 * pitch, (uint64_t)t->rows, 1};
        return tbh::encode_tiles_u4(map, t->codes, dims, strides, box, 128);
    }
    const uint64_t dims[3] = {pitch, (uint64_t)t->rows, 1};
    return tbh::encode_tiles_u8(map, t->codes, dims, strides, box, 128);
}

template <typename T, bool BOTH4>
int launch(const Args& a, const Plan& p, cudaStream_t s) {
    static std::atomic<uint64_t> granted{0};  // a bit per device
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    if (!(granted.load() >> ds->device & 1)) {
        TB_CUDA_TRY(cudaFuncSetAttribute(k_linear<T, BOTH4>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024));
        granted.fetch_or(1ull << ds->device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)p.bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_linear<T, BOTH4>, a));
    TB_LAUNCH_CHECK("microscaled product kernel");
    return TB_OK;
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
    rc = map_of(&a.w_map, w, kTileOuts, both4);
    if (rc == TB_OK) rc = map_of(&a.x_map, x, p.tile_rows, both4);
    if (rc != TB_OK) return rc;
    a.w_scales = w->scales;
    a.x_scales = x->scales;
    a.bias = bias;
    a.y = y;
    a.y_stride = y_stride;
    a.status = ds->status;
    a.rows = (int)x->rows;
    a.outs = (int)w->rows;
    a.tiles128 = (int)mx::tiles_of(x->cols);
    a.tile_rows = p.tile_rows;
    a.row_tiles = p.row_tiles;
    a.n_tiles = p.n_tiles;
    a.steps = p.steps;
    a.split = p.split;
    a.stages = p.stages;
    a.stage_bytes = p.stage_bytes;
    a.scales_off = p.scales_off;
    a.code_bytes = (kTileOuts >> (w->format == mx::kE2m1 && !both4)) * kStepBytes +
                   (p.tile_rows * kStepBytes >> (x->format == mx::kE2m1 && !both4));
    a.columns = p.columns;
    a.scales_column = p.scales_column;
    a.instruction = both4 ? tc::scaled_instruction_4bit()
                          : tc::scaled_instruction(element(w->format), element(x->format));
    cudaStream_t s = tbh::stream_of(stream);
    if (out_dtype == TB_DTYPE_F32)
        return both4 ? launch<float, true>(a, p, s) : launch<float, false>(a, p, s);
    return both4 ? launch<__nv_bfloat16, true>(a, p, s) : launch<__nv_bfloat16, false>(a, p, s);
}
