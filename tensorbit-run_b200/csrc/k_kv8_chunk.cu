// k_kv8_chunk.cu -- attention of many query rows (a chunk of a prompt) over the
// paged 8-bit cache: the mathematics of k_kv8_attention.cu with the products on
// the fifth-generation tensor cores.
//
// A CTA has 256 rows of one sequence and k/v head ((token, head of the group)
// pairs, token-major), as two tiles of 128, and walks their keys 128 at a time:
//   S = Q K^T  [128 x 128], operands f16 in shared memory, sums in tensor memory
//   P = 2^(S f - r), f16, over S's place in tensor memory
//   O += P V   P from tensor memory, V f16 in shared memory
// 4 warps bring codes by TMA, each its 32 keys, and write them as f16 tiles (two
// stages), 4 for each row tile compute P, a thread a row with its 128 scores in
// registers, and one warp issues the products, so that one tile's softmax runs
// while the other's products do.
//
// What bounds it, per 256 rows and 128 keys: the products, 4 * 128^3 at 4096 a
// clock, 2050 clocks; the exponentials, 32768 at 16 a clock, as many; converting
// 32768 codes, 7 % of the products' time an instruction.  Codes are converted
// once for 256 rows, four times fewer than a block of 16 rows' matrix
// instructions could share, and the products run at 4 times their rate.
//
// Measured: 2048 tokens behind 6144, 32 heads of 128 on 8, int8, 296 us, 812 TFLOP/s
// (0.49 of a library product's rate; blocks of 16 rows: 1634 us).  A step takes 2.35
// us, 4500 clocks: a tile's scores, softmax (2600) and products follow one another,
// and the products share shared memory's bandwidth with the conversion (3300 clocks
// where 2050 are the least).  256 CTAs of 49 to 64 steps, the longest first, give the
// busiest of 148 SMs 111 steps where 98 would be even shares: 0.88 full.  A CTA pays
// some 9 us beside its steps, so 64 sequences of 100 tokens and 1000 keys take 222 us
// (253 with a thread a row of q and out).  Keys are not cut: 100 rows of 64 heads on 8
// over 131071 keys are 32 CTAs of 1024 steps, 2.3 ms.
//
// Precision as in k_kv8_attention.cu: a row of q is scaled by a power of two to
// [2^14, 2^15) and held as f16, exact for bf16 elements above 2^-31 of the row's
// largest; weights are f16 times 2^11 under a reference r' that moves by whole
// powers of two; the values' scale joins the exponent, 2^(S f + log2 v_scale - r'
// + 11), and the sum of p takes each page's weights back to the row's r.  A page
// whose scale makes its weights less than 2^-100 of the row's largest adds to the
// sum alone: its f16 weights are zeros.
#include <math.h>

#include "kv8_mma.cuh"
#include "phases.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int kRows = 128;         // of a tile
constexpr int kTiles = 2;          // of a CTA
constexpr int kKeys = 128;         // of a step
constexpr int kGroups = kKeys / 16;  // of keys, each in one page
constexpr int kStages = 2;
using Stages = tbk::Ring<kStages>;
constexpr int kSoftWarps = 4 * kTiles, kConvWarps = 4;
constexpr int kIssuer = kSoftWarps + kConvWarps;  // the warp
constexpr int kThreads = 32 * (kIssuer + 4);  // a whole warpgroup, for its registers
// Registers a thread of each: 256 * 192 + 128 * 96 + 128 * 32 = 512 * 128 (with 184
// for the first 329 us where 192 took 308, with 72 and 56 for the others 301 where 96
// and 32 take 298).
constexpr int kSoftRegs = 192, kConvRegs = 96, kIssuerRegs = 32;
constexpr float kSlack = 4.0f, kLift = 11.0f, kLog2e = 1.4426950408889634f, kNoRef = -3.0e38f;
constexpr float kLeast = -100.0f;  // weights before the sum are at 2^kLeast of the row's or above
constexpr uint32_t kColumns = 512;  // of tensor memory: S and P at 0, 128, O at 256, 384

struct Args {
    CUtensorMap k_map, v_map;  // [n_pages * n_kv_heads][page][d] codes
    kv8::Batch b;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride;
    const float *k_scale, *v_scale;
    unsigned* status;
    float scale;
    int hq, hkv, d, window, max_rows, max_len, vec, vec_out;
};

template <int DP>
struct Shape {
    static constexpr int kPanels = DP / 64;
    static constexpr int kPanel = 128 * 128;  // bytes of 128 rows of 64 f16
    static constexpr int kTile = kPanels * kPanel;
    static constexpr int kCodes = 2 * kKeys * DP;  // a step's K and V as they are
    static constexpr int kBytes =
        kTiles * kTile + kStages * 2 * kTile + kCodes + 1024;  // 1024: to align
};

struct Shared {
    uint64_t k_full[kStages], v_full[kStages], kv_free[kStages];
    uint64_t s_full[kTiles], p_full[kTiles], o_done[kTiles];
    uint64_t codes[2][kConvWarps];  // of K, of V: the warp's have come
    uint64_t products_done;         // all that the issuer issued
    float2 scales[kStages][kGroups];  // of K (< 0: no page) and log2 of V's
    uint32_t tmem;
};

// Where the f16 element e of row r of a tile of 64-element panels lies.
__device__ __forceinline__ int place(int row, int piece) {  // 16-byte pieces of 8 elements
    return (piece >> 3) * (128 * 128) + row * 128 + ((piece ^ row) & 7) * 16;
}

// Two f32 at once.
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %4};\n"
        " mov.b64 c, {%5, %5};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Eight elements of a row, zeros if not live; vec: aligned to 16 bytes.
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, bool live, bool vec) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (live && vec) {
        x = *reinterpret_cast<const uint4*>(p);
    } else if (live) {
        const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) (&x.x)[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
    }
    return x;
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const uint4& x, bool vec) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = x;
    } else {
        uint16_t* u = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = (uint16_t)((&x.x)[i / 2] >> i % 2 * 16);
    }
}

// A bounded wait of a whole warp.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, unsigned* status) {
    const bool came = tbk::mbar_wait(bar, parity, status, 1000000000ull);
    return __all_sync(tbk::kFull, came);
}

template <int FORMAT>
__device__ __forceinline__ void to_f16(const uint4& codes, uint4 (&h)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (&codes.x)[i];
        uint32_t lo, hi;
        if constexpr (FORMAT == kv8::kInt8) {
            lo = kv8::int8_pair(kv8::prmt(w, 0, 0x4140));
            hi = kv8::int8_pair(kv8::prmt(w, 0, 0x4342));
        } else {
            lo = kv8::e4m3_pair(w, false);
            hi = kv8::e4m3_pair(w, true);
        }
        (&h[i / 2].x)[i % 2 * 2] = lo;
        (&h[i / 2].x)[i % 2 * 2 + 1] = hi;
    }
}

template <int FORMAT, int DP>
__global__ void __launch_bounds__(kThreads, 1) k_chunk(const __grid_constant__ Args a) {
    using H = Shape<DP>;
    using T = __nv_bfloat16;
    constexpr int kSteps = DP / 16;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared sh;
    uint8_t* smem = smem_raw + (-tbk::smem_addr(smem_raw) & 1023u);
    uint8_t* q_tiles = smem;
    uint8_t* kv_tiles = smem + kTiles * H::kTile;  // [stage][K, V]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A slot and head: sequence i's slots start at (its first row) / 256 + i, which is
    // one for each of its blocks or more; long blocks first.
    const int head = blockIdx.x % a.hkv, slot = (int)(gridDim.x - 1 - blockIdx.x) / a.hkv;
    const int group = a.hq / a.hkv;
    auto start = [&](int lo, int i) { return lo * group / (kTiles * kRows) + i; };
    kv8::Seq s;
    const int seq = kv8::find_sequence(a.b, slot, start, s);
    const int rows_all = s.n * group, block = slot - start(s.lo, seq);
    const int at = block * kTiles * kRows;
    if (block < 0 || at >= rows_all) return;
    const int rows = min(kTiles * kRows, rows_all - at);
    const int tiles = rows > kRows ? 2 : 1;
    const bool ok = s.len <= a.max_len && s.n <= a.max_rows &&
                    s.len <= ((int64_t)a.b.width << a.b.page_shift);
    if (!ok && threadIdx.x == 0) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
    // keys [seen, end) that some row sees, from a whole step
    const int p0 = s.first + at / group, p1 = s.first + (at + rows - 1) / group;
    const int end = ok ? max(p1 + 1, 0) : 0;
    const int seen = min(kv8::first_seen(p0, a.window), end), from = seen & ~(kKeys - 1);
    const int steps = (end - from + kKeys - 1) / kKeys;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tbk::mbar_init(&sh.k_full[i], kConvWarps);
            tbk::mbar_init(&sh.v_full[i], kConvWarps);
            tbk::mbar_init(&sh.kv_free[i], 1);
        }
        for (int i = 0; i < kTiles; ++i) {
            tbk::mbar_init(&sh.s_full[i], 1);
            tbk::mbar_init(&sh.p_full[i], 4);
            tbk::mbar_init(&sh.o_done[i], 1);
        }
        tbk::mbar_init(&sh.products_done, 1);
        for (int i = 0; i < kConvWarps; ++i) {
            tbk::mbar_init(&sh.codes[0][i], 1);
            tbk::mbar_init(&sh.codes[1][i], 1);
        }
        tbk::fence_mbar_init();
    }
    if (warp == kIssuer) tc::allocate(&sh.tmem, kColumns);

    // A converting warp has keys 32 w .. 32 w + 31 of each step, two groups of 16 whose
    // pages lanes 0 and 1 look up, ask for and ring in.
    const int32_t* table = a.b.table + seq * a.b.table_stride;
    const int first = from + 32 * (warp - kSoftWarps);  // its first key of step 0
    auto page_of = [&](int j) {  // lane's group's page of step j, -1 if none
        const int key = first + j * kKeys + 16 * lane;
        // (a page all in front of a window may be gone)
        if (lane > 1 || j >= steps || key >= end || key + 16 <= seen) return -1;
        const int id = table[key >> a.b.page_shift];
        if ((unsigned)id < (unsigned)a.b.n_pages) return id;
        atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
        return -1;
    };
    const bool converts = warp >= kSoftWarps && warp < kIssuer;
    int id = converts ? page_of(0) : -1, id_next = converts ? page_of(1) : -1;

    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = sh.tmem;

    // Q: a warp its 32 rows, all of them asked for at once, while the first codes
    // come; a lane has the 16-byte piece `piece` of every kRound-th row.  A row with a
    // NaN or an infinity is NaN.
    constexpr int kEach = DP / 8, kRound = 32 / kEach;
    const int tile = warp / 4, row0 = warp % 4 * 32, row = row0 + lane;
    const int piece = lane % kEach, r = tile * kRows + row;
    const bool soft = warp < kSoftWarps, live = soft && r < rows;
    float f = 0.0f;  // what the row's sums of products are multiplied with
    // where a row of the block stands in rows of `stride`, -1 if it is not there
    auto row_at = [&](int i, int64_t stride) {
        const int tok = i / group, h = head * group + i - tok * group;
        return live ? (s.lo + tok) * stride + (int64_t)h * a.d : (int64_t)-1;
    };
    if (soft && tile < tiles) {
        const int64_t mine = row_at(at + r, a.q_stride);
        uint4 x[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t there = __shfl_sync(tbk::kFull, mine, i * kRound + lane / kEach);
            x[i] = load8(static_cast<const T*>(a.q) + there + 8 * piece,
                         there >= 0 && 8 * piece < a.d, a.vec);
        }
        // the largest magnitudes of the even and of the odd elements: of piece i, then,
        // each lane keeping half of its rows, of all of row `piece` kRound + lane / kEach
        uint32_t two[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t m = 0x7fff7fffu;
            two[i] = __vmaxu2(__vmaxu2(x[i].x & m, x[i].y & m), __vmaxu2(x[i].z & m, x[i].w & m));
        }
#pragma unroll
        for (int o = kEach / 2; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < o; ++i) {
                const bool up = piece & o;
                const uint32_t other =
                    __shfl_xor_sync(tbk::kFull, up ? two[i] : two[i + o], o);
                two[i] = __vmaxu2(up ? two[i + o] : two[i], other);
            }
        const uint32_t top = max(two[0] & 0xffff0000u, two[0] << 16);
        const int e = min(max((int)(top >> 23), 1 + 16), 254);
        // a negative scale turns q, so that larger sums are larger scores
        const float lift = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23) *
                           (a.scale < 0.0f ? -1.0f : 1.0f);
        const float unit = top < 0x7f800000u ? __uint_as_float((uint32_t)(e - 14) << 23) *
                                                   (fabsf(a.scale) * kLog2e)
                                             : NAN;
        f = __shfl_sync(tbk::kFull, unit, lane % kRound * kEach + lane / kRound);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float by = __shfl_sync(tbk::kFull, lift, lane - piece + i);
            uint4 h;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = (&x[i].x)[j];
                (&h.x)[j] = kv8::pack_f16x2(__uint_as_float(w << 16) * by,
                                            __uint_as_float(w & 0xffff0000u) * by);
            }
            *reinterpret_cast<uint4*>(q_tiles + tile * H::kTile +
                                      place(row0 + i * kRound + lane / kEach, piece)) = h;
        }
        tbk::fence_proxy_async_shared();
    }

    if (warp >= kIssuer) {
        tc::fewer_registers<kIssuerRegs>();
        if (warp == kIssuer && steps > 0) {
            const bool leader = lane == 0;
            const uint32_t instr_s = tc::f16_instruction(kKeys, false);
            const uint32_t instr_o = tc::f16_instruction(DP, true);
            // descriptors count their start in units of 16 bytes
            const uint64_t q_desc = tc::tile_descriptor(tbk::smem_addr(q_tiles), 16);
            const uint64_t k_desc = tc::tile_descriptor(tbk::smem_addr(kv_tiles), 16);
            const uint64_t v_desc =
                tc::tile_descriptor(tbk::smem_addr(kv_tiles) + H::kTile, H::kPanel);
            auto scores = [&](int t, int j) {  // S of tile t and step j
                const uint64_t q = q_desc + t * (H::kTile / 16);
                const uint64_t k = k_desc + Stages::stage(j) * (2 * H::kTile / 16);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int off = (i / 4 * H::kPanel + i % 4 * 32) / 16;
                    tc::mma(tmem + t * 128, q + off, k + off, instr_s, i > 0, leader);
                }
                tc::commit(&sh.s_full[t], leader);
            };
            asm volatile("bar.sync 1, %0;" ::"n"(32 * (kSoftWarps + 1)) : "memory");  // Q
            bool fine = wait_all(&sh.k_full[0], 0, a.status);
            tc::fence_after();
            for (int t = 0; t < tiles && fine; ++t) scores(t, 0);
            for (int j = 0; j < steps && fine; ++j) {
                const int stage = Stages::stage(j);
                const uint64_t v = v_desc + stage * (2 * H::kTile / 16);
                fine = wait_all(&sh.v_full[stage], Stages::parity(j), a.status);
                for (int t = 0; t < tiles && fine; ++t) {
                    fine = wait_all(&sh.p_full[t], j & 1, a.status);
                    if (!fine) break;
                    tc::fence_after();
#pragma unroll
                    for (int i = 0; i < kKeys / 16; ++i)
                        tc::mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + i * 8,
                                     v + i * (2048 / 16), instr_o, j > 0 || i > 0, leader);
                    tc::commit(&sh.o_done[t], leader);
                    if (t == tiles - 1 && Stages::awaited(j, steps))
                        tc::commit(&sh.kv_free[stage], leader);
                    if (j + 1 < steps) {
                        if (t == 0) {
                            fine = wait_all(&sh.k_full[Stages::stage(j + 1)],
                                            Stages::parity(j + 1), a.status);
                            if (!fine) break;
                            tc::fence_after();
                        }
                        scores(t, j + 1);
                    }
                }
            }
            // whatever ended the loop, no product may be in flight when tensor memory is freed
            tc::commit(&sh.products_done, leader);
            wait_all(&sh.products_done, 0, a.status);
        }
    } else if (!soft) {
        tc::fewer_registers<kConvRegs>();
        // Codes to f16; a lane has the 16-byte piece c of every (32 / kWide)th key.
        constexpr int kWide = DP / 16, kStep = 32 / kWide;
        const int w = warp - kSoftWarps, c = lane % kWide;
        uint8_t* codes = kv_tiles + kStages * 2 * H::kTile + w * 2 * 32 * DP;  // K, V
        auto ask = [&](int kv, int j, int id) {  // the groups that have a page
            const uint32_t have = __ballot_sync(tbk::kFull, id >= 0);
            if (lane == 0 && have) tbk::mbar_expect_tx(&sh.codes[kv][w], __popc(have) * 16 * DP);
            __syncwarp();
            if (id >= 0) {
                const int slot = (first + j * kKeys + 16 * lane) & ((1 << a.b.page_shift) - 1);
                kv8::tma_load3(codes + (kv * 32 + 16 * lane) * DP, kv ? &a.v_map : &a.k_map, 0,
                               slot, id * a.hkv + head, &sh.codes[kv][w]);
            }
            return have;
        };
        uint32_t have_k = ask(0, 0, id), have_v = ask(1, 0, id);
        tbk::Phases phases;
        auto codes_came = [&](int kv) {
            return phases.wait(
                kv, [&](uint32_t parity) { return wait_all(&sh.codes[kv][w], parity, a.status); });
        };
        float2 scale = make_float2(-1.0f, 0.0f);
        auto ask_scale = [&] {
            scale = make_float2(-1.0f, 0.0f);
            if (id >= 0)
                scale = make_float2(a.k_scale[id * a.hkv + head], a.v_scale[id * a.hkv + head]);
        };
        ask_scale();
        bool fine = true;
        for (int j = 0; j < steps && fine; ++j) {
            const int stage = Stages::stage(j), key0 = first + j * kKeys;
            fine = !Stages::reused(j) ||
                   wait_all(&sh.kv_free[stage], Stages::parity(j - kStages), a.status);
            if (!fine) break;
            uint8_t* to = kv_tiles + stage * 2 * H::kTile;
            if (lane < 2)
                sh.scales[stage][2 * w + lane] = make_float2(
                    scale.x, (float)((int)(__float_as_uint(scale.y) >> 23) - 127));
            id = id_next;
            id_next = page_of(j + 2);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const uint32_t have = kv ? have_v : have_k;
                fine = !have || codes_came(kv);
                if (!fine) break;
                uint4 x[kWide];
#pragma unroll
                for (int i = 0; i < kWide; ++i)
                    x[i] = *reinterpret_cast<const uint4*>(
                        codes + (kv * 32 + lane / kWide + i * kStep) * DP + c * 16);
                if (have != 3 || key0 < seen || key0 + 32 > end) {
                    // slots of no page or that no row of the block sees may hold anything
#pragma unroll
                    for (int i = 0; i < kWide; ++i) {
                        const int key = lane / kWide + i * kStep;
                        if (!(have >> key / 16 & 1) || key0 + key < seen || key0 + key >= end)
                            x[i] = make_uint4(0, 0, 0, 0);
                    }
                }
                // all lanes have their codes: the next step's may come
                tbk::fence_proxy_async_shared();
                __syncwarp();
                (kv ? have_v : have_k) = ask(kv, j + 1, id);
#pragma unroll
                for (int i = 0; i < kWide; ++i) {
                    uint4 h[2];
                    to_f16<FORMAT>(x[i], h);
                    // the lanes of a key's second panel write their pieces in the
                    // other order, into other banks
                    const int key = 32 * w + lane / kWide + i * kStep, y = c >> 2;
                    uint8_t* tile_at = to + kv * H::kTile;
                    *reinterpret_cast<uint4*>(tile_at + place(key, 2 * c + y)) = y ? h[1] : h[0];
                    *reinterpret_cast<uint4*>(tile_at + place(key, 2 * c + 1 - y)) =
                        y ? h[0] : h[1];
                }
                tbk::fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0) tbk::mbar_arrive(kv ? &sh.v_full[stage] : &sh.k_full[stage]);
            }
            ask_scale();
        }
        if (!fine) {  // no copy may be in flight when the block ends
            if (have_k) codes_came(0);
            if (have_v) codes_came(1);
        }
    } else {
        if (steps > 0) asm volatile("bar.arrive 1, %0;" ::"n"(32 * (kSoftWarps + 1)) : "memory");
        tc::more_registers<kSoftRegs>();
        if (tile < tiles) {
        const uint32_t s_at = tmem + tile * 128 + ((uint32_t)(warp % 4) << 21);
        const uint32_t o_at = s_at + 256;
        const int see_hi = live ? s.first + (at + r) / group : INT32_MAX;
        // a row before position 0 sees no key, so that a see_lo that wraps does no harm
        const int see_lo =
            live && a.window ? max((int)((unsigned)see_hi - (unsigned)a.window + 1u), 0) : 0;
        float ref = kNoRef, vref = kNoRef, sum = 0.0f;
        bool fine = true;
        for (int j = 0; j < steps; ++j) {
            fine = wait_all(&sh.k_full[Stages::stage(j)], Stages::parity(j), a.status) &&
                   wait_all(&sh.s_full[tile], j & 1, a.status);
            if (!fine) break;
            tc::fence_after();
            const int key0 = from + j * kKeys;
            float fs[kGroups], lv[kGroups];
            uint32_t have = 0;  // groups that have a page
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float2 x = sh.scales[Stages::stage(j)][i];
                fs[i] = f * x.x;
                lv[i] = x.y;
                have |= (uint32_t)!(x.x < 0.0f) << i;
            }
            const bool inside =
                __all_sync(tbk::kFull, key0 >= see_lo && key0 + kKeys - 1 <= see_hi &&
                                           have == (1u << kGroups) - 1);
            // sums of products, or, of a step with keys that a row does not see, scores
            float x[kKeys];
            tc::load<kKeys>(s_at, x);
            if (!inside) {
#pragma unroll
                for (int e = 0; e < kKeys; ++e) {
                    const bool seen = key0 + e >= see_lo && key0 + e <= see_hi && (have >> e / 16 & 1);
                    x[e] = seen ? x[e] * fs[e / 16] : -INFINITY;
                }
            }
            // the largest score, and with the values' scale
            float hi = -INFINITY, hv = -INFINITY;
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                float m = max3(x[16 * i], x[16 * i + 1], x[16 * i + 2]);
#pragma unroll
                for (int e = 3; e < 15; e += 2) m = max3(m, x[16 * i + e], x[16 * i + e + 1]);
                m = fmaxf(m, x[16 * i + 15]);
                if (inside) m *= fs[i];
                hi = fmaxf(hi, m);
                hv = fmaxf(hv, m + lv[i]);
            }
            const bool over = hi > ref + kSlack || hv > vref + kSlack;
            if (__any_sync(tbk::kFull, over)) {
                const float m = over ? fmaxf(ref, ceilf(hi)) : ref;
                const float mv = over ? fmaxf(vref, ceilf(hv)) : vref;
                sum *= exp2f(ref - m);
                if (__any_sync(tbk::kFull, mv > vref) && j > 0) {
                    // O is free between its products of two steps
                    fine = wait_all(&sh.o_done[tile], (j - 1) & 1, a.status);
                    if (!fine) break;
                    tc::fence_after();
                    const float keep = exp2f(vref - mv);
#pragma unroll 1
                    for (int c0 = 0; c0 < DP; c0 += 32) {
                        float o[32];
                        tc::load<32>(o_at + c0, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= keep;
                        tc::store32(o_at + c0, o);
                    }
                    tc::wait_store();
                }
                ref = m;
                vref = mv;
            }
            // weights times the values' scale; a group's sum back without it
            const float least = kLeast - ref, shift = kLift - vref;
#pragma unroll
            for (int c0 = 0; c0 < kKeys; c0 += 32) {
                uint32_t p[16];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int i = c0 / 16 + g;
                    const float up = fmaxf(lv[i] + shift, least);
                    const float fi = inside ? fs[i] : 1.0f;
                    float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float2 y = fma2(make_float2(x[16 * i + e], x[16 * i + e + 1]), fi, up);
                        y.x = kv8::exp2_fast(y.x);
                        y.y = kv8::exp2_fast(y.y);
                        part = add2(part, y);
                        p[8 * g + e / 2] = kv8::pack_f16x2(y.x, y.y);
                    }
                    sum = fmaf(part.x + part.y, kv8::exp2_fast(-up - ref), sum);
                }
                tc::store16(s_at + c0 / 2, p);
            }
            tc::wait_store();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tbk::mbar_arrive(&sh.p_full[tile]);
        }
        if (fine && steps > 0) fine = wait_all(&sh.o_done[tile], (steps - 1) & 1, a.status);
        tc::fence_after();
        const bool none = !(sum != 0.0f);
        const float per = none || !fine ? 0.0f : exp2f(vref - ref - kLift) / sum;
        // through the rows of Q that are its own, for whole rows to be stored at once
        uint8_t* own = q_tiles + tile * H::kTile;
#pragma unroll 1
        for (int c0 = 0; c0 < DP; c0 += 32) {
            float x[32];
            if (steps > 0) tc::load<32>(o_at + c0, x);
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = none || steps == 0 ? 0.0f : x[e + i] * per;
                *reinterpret_cast<uint4*>(own + place(row, (c0 + e) / 8)) =
                    make_uint4(tbk::pack_bf16x2(y[0], y[1]), tbk::pack_bf16x2(y[2], y[3]),
                               tbk::pack_bf16x2(y[4], y[5]), tbk::pack_bf16x2(y[6], y[7]));
            }
        }
        __syncwarp();
        const int64_t mine = row_at(at + r, a.out_stride);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int other = i * kRound + lane / kEach;
            const int64_t there = __shfl_sync(tbk::kFull, mine, other);
            const uint4 y = *reinterpret_cast<const uint4*>(own + place(row0 + other, piece));
            if (there >= 0 && 8 * piece < a.d)
                store8(static_cast<T*>(a.out) + there + 8 * piece, y, a.vec_out);
        }
        if (a.lse && live)
            a.lse[(int64_t)(s.lo + (at + r) / group) * a.hq + head * group + (at + r) % group] =
                none ? -INFINITY : ref * 0.69314718055994531f + logf(sum);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == kIssuer) tc::release(tmem, kColumns);
}

template <int FORMAT, int DP>
int launch(Args& a, const TbB200Kv8* cache, dim3 grid, cudaStream_t s) {
    constexpr int bytes = Shape<DP>::kBytes;
    static std::atomic<uint64_t> granted{0};  // a bit per device
    int rc = kv8::once_per_device(granted, [&] {
        return cudaFuncSetAttribute(k_chunk<FORMAT, DP>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    });
    if (rc == TB_OK) rc = kv8::tile_map(&a.k_map, cache, cache->k, DP, 16, false);
    if (rc == TB_OK) rc = kv8::tile_map(&a.v_map, cache, cache->v, DP, 16, false);
    if (rc != TB_OK) return rc;
    k_chunk<FORMAT, DP><<<grid, kThreads, bytes, s>>>(a);
    TB_LAUNCH_CHECK("8-bit cache chunk attention kernel");
    return TB_OK;
}

// Slots of the grid: a bound on the batch's blocks, whatever max_rows is (64 sequences
// of 100 rows took 253 us; with a grid of max_rows for each, 245 if that is 100 and
// 545 if it is the batch's 6400).
int64_t slots_of(const TbB200Kv8* cache, const TbB200Kv8Batch* batch,
                 const TbB200Kv8Attention* t) {
    const int64_t group = t->n_heads / cache->n_kv_heads;
    return batch->rows * group / (kTiles * kRows) + batch->n_seqs;
}

}  // namespace

namespace kv8 {

// A wave of this kernel's CTAs takes a step of 128 keys in about 2.35 us (1.95 with
// heads of 64) however few of their rows are there, k_attend the same keys in 6.6 ns
// (3.9) for each block of 16 rows, so one wave is worth 356 (500) blocks, 2.4 (3.4, of
// which the rule takes 3.3) for each of 148 SMs.  The rule is for a whole call, by its
// bounds, and both sides were measured on equal sequences: a prompt beside single
// tokens takes this kernel for all of them (2048 rows beside 63 single tokens of up to
// 8191 keys, 64 heads on 8: 361 us, where a call for each kind takes 120 and 91).
// Both sides, this kernel's first, 32 heads of 128 on 8, int8, 2048 keys: one
// sequence of 160 rows 55 and 56 us, 256 55 and 78, 512 55 and 135; 16 of 8 rows 45
// and 44, 16 of 16 46 and 76; 64 of 8 167 and 136, 64 of 12 169 and 197.  Heads of
// 64, e4m3: one of 160 46 and 42, 256 44 and 54; 64 of 12 142 and 114, 16 141 and 146.
bool chunk_suits(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
                 int sm_count) {
    if (t->dtype != TB_DTYPE_BF16 || cache->head_dim > 128) return false;
    const int64_t group = t->n_heads / cache->n_kv_heads, rows = batch->rows * group;
    const int64_t slots = slots_of(cache, batch, t);
    const int64_t most = t->max_rows < batch->rows ? t->max_rows : batch->rows;
    const int64_t each = (most * group + kTiles * kRows - 1) / (kTiles * kRows) * batch->n_seqs;
    const int64_t waves =
        ((each < slots ? each : slots) * cache->n_kv_heads + sm_count - 1) / sm_count;
    if (slots * cache->n_kv_heads > INT32_MAX) return false;
    const double small = (double)rows * cache->n_kv_heads / 16;
    return small >= (cache->head_dim <= 64 ? 3.3 : 2.4) * (double)(waves * sm_count);
}

int chunk_attention(const TbB200Kv8* cache, const TbB200Kv8Batch* batch,
                    const TbB200Kv8Attention* t, cudaStream_t stream) {
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    Args a = {};
    a.b = view(cache, batch);
    a.q = t->q;
    a.out = t->out;
    a.lse = t->lse;
    a.q_stride = t->q_stride;
    a.out_stride = t->out_stride;
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.status = ds->status;
    a.scale = t->scale;
    a.hq = t->n_heads;
    a.hkv = cache->n_kv_heads;
    a.d = cache->head_dim;
    a.window = t->window;
    a.max_rows = t->max_rows;
    a.max_len = t->max_len;
    a.vec = tbh::aligned16(t->q) && t->q_stride % 8 == 0;
    a.vec_out = tbh::aligned16(t->out) && t->out_stride % 8 == 0;
    const dim3 grid((unsigned)(slots_of(cache, batch, t) * a.hkv));
    const bool int8 = cache->format == kInt8;
    if (cache->head_dim <= 64)
        return int8 ? launch<kInt8, 64>(a, cache, grid, stream)
                    : launch<kE4m3, 64>(a, cache, grid, stream);
    return int8 ? launch<kInt8, 128>(a, cache, grid, stream)
                : launch<kE4m3, 128>(a, cache, grid, stream);
}

}  // namespace kv8
