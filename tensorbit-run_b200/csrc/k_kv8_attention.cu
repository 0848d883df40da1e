// k_kv8_attention.cu -- attention of Q rows over the paged 8-bit cache.
//
//   s_j = scale q.k_j,  out = sum_j p_j v_j,  p = softmax(s),  k_j = code * page scale
//
// A block holds 16 rows of one sequence and k/v head: (query token, head of the
// group) pairs, token-major.  With a group of 8 heads and one token half of
// them are empty, which costs nothing while the cache's bytes bound the time.
// Its keys are split into chunks over CTAs when there are few blocks; a second
// kernel joins the chunks.
//
// Within a CTA each of 4 warps takes every fourth step of 16 keys, which lie in
// one page, through a ring of cp.async stages of its own: no barrier in the
// loop.  The codes go from shared memory to registers with 16-byte loads and
// are converted there, each lane having exactly the operands of its m16n8k16
// instructions:
//   S = Q K^T: lane (g, t) (g = lane / 4, t = lane % 4) holds key order(g), 16
//     consecutive elements of it; a word's even and odd bytes are the two
//     operand registers of one 16-wide step, so the head dimension is summed
//     in the order that Q's registers are laid out in too;
//   O = P V: S's registers are P's operands; lane (g, t) holds the elements
//     16 g .. 16 g + 15 (of 128) of keys order(2t), order(2t + 1).
// order() and the two swizzles below put the 8 lanes of each 16-byte access
// into different banks.
//
// Precision.  A code is an f16 exactly.  A row of q is scaled by a power of two
// to [2^14, 2^15) and held as f16: bf16 elements exactly unless 2^-21 below the
// row's largest, where what is lost is 2^-39 of the largest; f32 rows as two f16 (hi + lo), 22 bits.
// Weights p are f16 relative to a power of two near the row's largest (half a
// step 2^-12, an eighth of the bf16 output's), for f32 rows hi + lo again.
// Sums, maxima and the sum of p are f32.  The values' scale joins the exponent,
// p v_scale = 2^(s + log2 v_scale - r'), with a reference r' of its own per
// row, so pages of any scales keep their weight.  References are whole numbers
// and move only when a score passes them by 2^4: rescaling is exact and rare.
// A weight more than 2^-25 below the row's largest is an f16 subnormal, off by
// at most 2^-36 of the largest.
#include "kv8_mma.cuh"
#include "tma.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;          // keys a warp takes at once
constexpr int kLeastChunk = 256;   // keys below which a chunk is not split further
constexpr float kSlack = 4.0f;     // how far (log2) scores may pass a reference
constexpr float kLift = 11.0f;     // weights are held times 2^11: up to 2^15 in f16
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    kv8::Batch b;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    unsigned* status;
    float* part;    // [seq, kv head, block, chunk][16][d] partial outputs
    float2* state;  // the same [16]: (reference, sum)
    float scale;
    int hq, hkv, d, window, max_rows, max_len, chunks, blocks, vec;
};

// What a block of 16 rows attends, the same in both kernels.
struct Block {
    kv8::Seq s;
    int rows;       // live rows of the block
    int lo, end;    // keys [lo, end) that some row sees
    int from, size; // chunk c: keys [from + c size, from + (c + 1) size)
    int used;       // chunks that are not empty (1 if no key at all)
};

__device__ __forceinline__ Block block_of(const Args& a, int seq, int block, bool flag) {
    Block k;
    k.s = kv8::sequence(a.b, seq);
    const int group = a.hq / a.hkv;
    const int64_t all = (int64_t)k.s.n * group, at = (int64_t)block * 16;
    k.rows = (int)max((int64_t)0, min((int64_t)16, all - at));
    k.lo = k.end = 0;
    if (k.rows > 0) {
        if (k.s.len > a.max_len || k.s.n > a.max_rows ||
            k.s.len > ((int64_t)a.b.width << a.b.page_shift)) {
            if (flag) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
        } else {
            const int p0 = k.s.first + (int)(at / group);
            const int p1 = k.s.first + (int)((at + k.rows - 1) / group);
            k.end = max(p1 + 1, 0);
            k.lo = a.window ? min(max(p0 - a.window + 1, 0), k.end) : 0;
        }
    }
    k.from = k.lo & ~(kStep - 1);
    const int keys = k.end - k.from;
    const int each = (keys + a.chunks - 1) / a.chunks;
    k.size = max(kLeastChunk, (each + kWarps * kStep - 1) / (kWarps * kStep) * (kWarps * kStep));
    k.used = max(1, (keys + k.size - 1) / k.size);
    return k;
}

// The key of a step that column (or lane group) n of 8 stands for.
__device__ __forceinline__ int order(int n) { return n & 1 ? (n >> 1) ^ 5 : n >> 1; }
// Where a row's 16-byte piece c lies.
__device__ __forceinline__ int k_place(int key, int c, int pieces) {
    return pieces > 4 ? c ^ ((key & 1) << 2) : c;
}
__device__ __forceinline__ int v_place(int key, int c, int pieces) {
    return pieces > 4 ? c ^ ((key & 3) << 1) : c ^ (key & 2);
}

template <int DP>
constexpr int stages() {
    return DP == 64 ? 6 : DP == 128 ? 4 : 3;
}
template <int DP>
constexpr int stage_bytes() {
    return 2 * kStep * DP;
}
// Q's operands stay in registers when they are few.
template <typename T, int DP>
constexpr bool q_in_registers() {
    return DP / 16 * 4 * (sizeof(T) == 4 ? 2 : 1) <= 32;
}
template <typename T, int DP>
constexpr int smem_bytes() {
    const int ring = kWarps * stages<DP>() * (stage_bytes<DP>() + 16);
    const int q = q_in_registers<T, DP>() ? 0 : DP / 16 * 512 * (sizeof(T) == 4 ? 2 : 1);
    const int join = kWarps * 16 * (DP + 4) * 4 + kWarps * 16 * 12;
    return (ring > join ? ring : join) + q;
}

template <typename T, int FORMAT, int DP>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 2 : 3)
k_attend(const __grid_constant__ Args a) {
    constexpr bool kSplit = sizeof(T) == 4;   // hi + lo operands
    constexpr bool kQReg = q_in_registers<T, DP>();
    constexpr int kSteps = DP / 16;           // 16-wide steps of the head dimension
    constexpr int kStages = stages<DP>();
    constexpr int kPieces = DP / 16;          // 16-byte pieces of a key
    constexpr int kOut = DP / 8;              // 8-wide output tiles
    extern __shared__ __align__(16) uint8_t smem[];

    const int c = blockIdx.x % a.chunks, block = blockIdx.x / a.chunks;
    const int head = blockIdx.y, seq = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Block blk = block_of(a, seq, block, threadIdx.x == 0 && c == 0 && head == 0);
    if (blk.rows == 0 || c >= blk.used) return;
    const int group = a.hq / a.hkv;
    const int begin = blk.from + c * blk.size, end = min(begin + blk.size, blk.end);

    // the two rows of this lane: keys [see_lo, see_hi] each
    int see_lo[2], see_hi[2];
    float qf[2];  // what a row's scores are multiplied with, but for the page's scale
    uint32_t qr[kQReg ? kSteps : 1][4], ql[kQReg && kSplit ? kSteps : 1][4];
    uint4* qs = reinterpret_cast<uint4*>(
        smem + (smem_bytes<T, DP>() - (kQReg ? 0 : kSteps * 512 * (kSplit ? 2 : 1))));
    {
        const T* qp[2];
        float top[2] = {0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int i = g + 8 * r;
            const bool live = i < blk.rows;
            const int64_t at = (int64_t)block * 16 + i;
            const int tok = live ? (int)(at / group) : 0, hh = live ? (int)(at % group) : 0;
            // rows of the block that are not there see all and are not stored
            const int p = live ? blk.s.first + tok : INT32_MAX;
            see_hi[r] = p;
            see_lo[r] = a.window && live ? max(p - a.window + 1, 0) : 0;
            qp[r] = live ? static_cast<const T*>(a.q) + (blk.s.lo + tok) * a.q_stride +
                               (int64_t)(head * group + hh) * a.d
                         : nullptr;
            if (live) {
#pragma unroll
                for (int h = 0; h < DP / 64; ++h) {
                    float x[16];
                    kv8::load16(qp[r] + 64 * h + 16 * t, 64 * h + 16 * t < a.d, a.vec, x);
#pragma unroll
                    for (int e = 0; e < 16; ++e) top[r] = fmaxf(top[r], fabsf(x[e]));
                }
            }
            top[r] = fmaxf(top[r], __shfl_xor_sync(tbk::kFull, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(tbk::kFull, top[r], 2));
        }
        float lift[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            // 2^e with |q| 2^e in [2^14, 2^15); NaN and infinite rows stay that
            const int e = min(max((int)(__float_as_uint(top[r]) >> 23), 1 + 16), 254);
            lift[r] = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23);
            qf[r] = __uint_as_float((uint32_t)(e - 14) << 23) * (a.scale * kLog2e) *
                    kv8::kOperandUnit<FORMAT>;
        }
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) {
            float x[2][16];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                kv8::load16(qp[r] + 64 * h + 16 * t, qp[r] && 64 * h + 16 * t < a.d, a.vec, x[r]);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[r][e] *= lift[r];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // a word of 4 codes: even ones, odd ones
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float u = x[r][4 * j + e], w = x[r][4 * j + e + 2];
                        hi[2 * e + r] = kv8::pack_f16x2(u, w);
                        const __half2 h2 = *reinterpret_cast<const __half2*>(&hi[2 * e + r]);
                        lo[2 * e + r] =
                            kv8::pack_f16x2(u - __low2float(h2), w - __high2float(h2));
                    }
                const int s = 4 * h + j;
                if constexpr (kQReg) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        qr[s][e] = hi[e];
                        if (kSplit) ql[s][e] = lo[e];
                    }
                } else if (warp == 0) {
                    qs[s * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (kSplit) qs[(kSteps + s) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        }
    }
    if constexpr (!kQReg) __syncthreads();

    // the warp's steps: keys first + 64 n .. + 15
    const int first = begin + warp * kStep;
    const int n_steps = end > first ? (end - first + kWarps * kStep - 1) / (kWarps * kStep) : 0;
    uint8_t* ring = smem + warp * kStages * (stage_bytes<DP>() + 16);
    const uint32_t ring_s = tbk::smem_addr(ring);
    const int32_t* table = a.b.table + seq * a.b.table_stride;
    const int pieces = a.d / 16;
    auto page_of = [&](int n) {  // the page of step n, -1 if it has none
        if (n >= n_steps) return -1;
        const int id = table[(first + n * (kWarps * kStep)) >> a.b.page_shift];
        if (id >= 0 && id < a.b.n_pages) return id;
        atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
        return -1;
    };
    int ids = page_of(lane), ids_next = page_of(32 + lane);  // of steps [0, 32), [32, 64)
    auto issue = [&](int n) {
        const int id = __shfl_sync(tbk::kFull, ids, n & 31);
        if ((n & 31) == 31) {
            ids = ids_next;
            ids_next = page_of(n + 33 + lane);
        }
        if (id >= 0) {
            const int64_t unit = (int64_t)id * a.hkv + head;
            const int slot = (first + n * (kWarps * kStep)) & ((1 << a.b.page_shift) - 1);
            const int64_t at = ((unit << a.b.page_shift) + slot) * a.d;
            const uint32_t dst = ring_s + (n % kStages) * (stage_bytes<DP>() + 16);
            constexpr int kRows = 32 / kPieces > 0 ? 32 / kPieces : 1;  // keys per warp access
            const int piece = lane % kPieces;
            if (piece < pieces) {
#pragma unroll
                for (int i = 0; i < kStep / kRows; ++i) {
                    const int key = lane / kPieces + i * kRows;
                    const int64_t from = at + key * a.d + piece * 16;
                    const uint32_t row = dst + key * DP;
                    kv8::cp_async16(row + k_place(key, piece, kPieces) * 16, a.k + from);
                    kv8::cp_async16(row + kStep * DP + v_place(key, piece, kPieces) * 16,
                                    a.v + from);
                }
            }
            if (lane < 2)
                kv8::cp_async4(dst + stage_bytes<DP>() + 4 * lane,
                               (lane ? a.v_scale : a.k_scale) + unit);
        }
        const bool there = id >= 0;
        kv8::cp_async_commit();
        return there;
    };
    uint32_t there = 0;  // bit i: the step i behind the newest issued one has a page
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) there = there << 1 | (uint32_t)issue(n);

    float o[kOut][4];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float ref[2] = {-INFINITY, -INFINITY}, vref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

    for (int n = 0; n < n_steps; ++n) {
        kv8::cp_async_wait<kStages - 2>();
        __syncwarp();
        there = there << 1 | (uint32_t)issue(n + kStages - 1);
        if (!(there >> (kStages - 1) & 1)) continue;
        const uint8_t* stage = ring + (n % kStages) * (stage_bytes<DP>() + 16);
        const float2 scales = *reinterpret_cast<const float2*>(stage + stage_bytes<DP>());
        const int key0 = first + n * (kWarps * kStep);

        // S: two tiles of 8 keys
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
            const int key = 8 * i + order(g);
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) {
                const uint4 w4 = *reinterpret_cast<const uint4*>(
                    stage + key * DP + k_place(key, 4 * h + t, kPieces) * 16);
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t b0, b1;
                    kv8::to_f16<FORMAT>(w[j], b0, b1);
                    const int k = 4 * h + j;
                    if constexpr (kQReg) {
                        kv8::mma16816(s[i], qr[k][0], qr[k][1], qr[k][2], qr[k][3], b0, b1);
                        if constexpr (kSplit)
                            kv8::mma16816(s[i], ql[k][0], ql[k][1], ql[k][2], ql[k][3], b0, b1);
                    } else {
                        const uint4 x = qs[k * 32 + lane];
                        kv8::mma16816(s[i], x.x, x.y, x.z, x.w, b0, b1);
                        if constexpr (kSplit) {
                            const uint4 y = qs[(kSteps + k) * 32 + lane];
                            kv8::mma16816(s[i], y.x, y.y, y.z, y.w, b0, b1);
                        }
                    }
                }
            }
        }
        // log2 units; the values' scale as an exponent
        const float lv = (float)((int)(__float_as_uint(scales.y) >> 23) - 127);
        bool over = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float f = qf[r] * scales.x;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) s[i][2 * r + e] *= f;
        }
        const bool inside = key0 >= see_lo[0] && key0 >= see_lo[1] &&
                            key0 + kStep - 1 <= see_hi[0] && key0 + kStep - 1 <= see_hi[1];
        if (!__all_sync(tbk::kFull, inside)) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = key0 + 8 * i + order(2 * t + (e & 1));
                    if (j < see_lo[e >> 1] || j > see_hi[e >> 1]) s[i][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float hi = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]),
                                   fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            over |= hi > ref[r] + kSlack || hi + lv > vref[r] + kSlack;
        }
        if (__any_sync(tbk::kFull, over)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float hi = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]),
                                 fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                hi = fmaxf(hi, __shfl_xor_sync(tbk::kFull, hi, 1));
                hi = fmaxf(hi, __shfl_xor_sync(tbk::kFull, hi, 2));
                const float m = fmaxf(ref[r], ceilf(hi)), mv = fmaxf(vref[r], ceilf(hi) + lv);
                if (m > ref[r]) sum[r] *= kv8::exp2_fast(ref[r] - m);
                if (mv > vref[r]) {
                    const float keep = kv8::exp2_fast(vref[r] - mv);
#pragma unroll
                    for (int i = 0; i < kOut; ++i) {
                        o[i][2 * r] *= keep;
                        o[i][2 * r + 1] *= keep;
                    }
                }
                ref[r] = m;
                vref[r] = mv;
            }
        }
        // weights: for the sum, and times the values' scale as P's operands
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float m = ref[r] == -INFINITY ? 0.0f : ref[r];
            const float mv = (vref[r] == -INFINITY ? 0.0f : vref[r]) - lv - kLift;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float s0 = s[i][2 * r], s1 = s[i][2 * r + 1];
                sum[r] += kv8::exp2_fast(s0 - m) + kv8::exp2_fast(s1 - m);
                const float p0 = kv8::exp2_fast(s0 - mv), p1 = kv8::exp2_fast(s1 - mv);
                ph[2 * i + r] = kv8::pack_f16x2(p0, p1);
                if constexpr (kSplit) {
                    const __half2 h2 = *reinterpret_cast<const __half2*>(&ph[2 * i + r]);
                    pl[2 * i + r] = kv8::pack_f16x2(p0 - __low2float(h2), p1 - __high2float(h2));
                }
            }
        }
        // O += P V
        const uint8_t* vs = stage + kStep * DP;
        const int ka = order(2 * t), kb = order(2 * t + 1);
        constexpr int kWide = DP >= 128 ? 16 : 8;  // bytes a lane takes of a key at once
#pragma unroll
        for (int h = 0; h < (DP + 127) / 128; ++h) {
            uint32_t w[4][kWide / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = (i & 1 ? kb : ka) + (i & 2 ? 8 : 0);
                const uint8_t* row = vs + key * DP;
                if constexpr (DP >= 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(
                        row + v_place(key, 8 * h + g, kPieces) * 16);
                    w[i][0] = x.x;
                    w[i][1] = x.y;
                    w[i][2] = x.z;
                    w[i][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(
                        row + v_place(key, g >> 1, kPieces) * 16 + (g & 1) * 8);
                    w[i][0] = x.x;
                    w[i][1] = x.y;
                }
            }
#pragma unroll
            for (int j = 0; j < kWide / 4; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t sel = half ? 0x7632 : 0x5410;
                    uint32_t b0e, b0o, b1e, b1o;
                    kv8::to_f16<FORMAT>(kv8::prmt(w[0][j], w[1][j], sel), b0e, b0o);
                    kv8::to_f16<FORMAT>(kv8::prmt(w[2][j], w[3][j], sel), b1e, b1o);
                    const int tile = h * 16 + 4 * j + 2 * half;
                    kv8::mma16816(o[tile], ph[0], ph[1], ph[2], ph[3], b0e, b1e);
                    kv8::mma16816(o[tile + 1], ph[0], ph[1], ph[2], ph[3], b0o, b1o);
                    if constexpr (kSplit) {
                        kv8::mma16816(o[tile], pl[0], pl[1], pl[2], pl[3], b0e, b1e);
                        kv8::mma16816(o[tile + 1], pl[0], pl[1], pl[2], pl[3], b0o, b1o);
                    }
                }
        }
    }
    kv8::cp_async_wait<0>();
    __syncthreads();  // the rings are free: the warps' states meet in their place

    // lane (g, t) has columns 2t, 2t + 1 of each tile: element (2t + e) * kWide + tile
    constexpr int kPitch = DP + 4;
    float* jo = reinterpret_cast<float*>(smem);
    float* jm = jo + kWarps * 16 * kPitch;
    constexpr int kWide = DP >= 128 ? 16 : 8;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        sum[r] += __shfl_xor_sync(tbk::kFull, sum[r], 1);
        sum[r] += __shfl_xor_sync(tbk::kFull, sum[r], 2);
        float* row = jo + (warp * 16 + g + 8 * r) * kPitch;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                row[(i / kWide) * 128 + (2 * t + e) * kWide + i % kWide] = o[i][2 * r + e];
        if (t == 0) {
            float* st = jm + (warp * 16 + g + 8 * r) * 3;
            st[0] = ref[r];
            st[1] = vref[r];
            st[2] = sum[r];
        }
    }
    __syncthreads();
    const bool whole = blk.used == 1;
    const int64_t unit =
        (((int64_t)seq * a.hkv + head) * a.blocks + block) * a.chunks + c;
    for (int row = warp; row < blk.rows; row += kWarps) {
        float m = -INFINITY, mv = -INFINITY, total = 0.0f, w[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            m = fmaxf(m, jm[(i * 16 + row) * 3]);
            mv = fmaxf(mv, jm[(i * 16 + row) * 3 + 1]);
        }
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float* st = jm + (i * 16 + row) * 3;
            total += st[0] == -INFINITY ? st[2] : st[2] * exp2f(st[0] - m);
            w[i] = st[1] == -INFINITY ? 0.0f : exp2f(st[1] - mv);
        }
        const bool none = total == 0.0f;
        // O is in units of 2^(mv - lift); of the sum's 2^m
        const float per = none ? 0.0f
                               : kv8::kOperandUnit<FORMAT> * exp2f(-kLift) / total;
        const float unit_v = none ? 0.0f : exp2f(mv - m);
        const int64_t at = (int64_t)block * 16 + row;
        const int64_t tok = blk.s.lo + at / group;
        const int h = head * group + (int)(at % group);
        T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
        float* part = whole ? nullptr : a.part + (unit * 16 + row) * a.d;
        for (int i = lane; i < a.d; i += 32) {
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) y += w[k] * jo[(k * 16 + row) * kPitch + i];
            y = none ? 0.0f : y * per * unit_v;
            if (whole)
                tbk::Elt<T>::store(out + i, y);
            else
                part[i] = y;
        }
        if (lane == 0) {
            if (!whole)
                a.state[unit * 16 + row] = make_float2(m, total);
            else if (a.lse)
                a.lse[tok * a.hq + h] = none ? -INFINITY : m * 0.69314718055994531f + logf(total);
        }
    }
}

// Joins the chunks of each block: out = sum_c w_c out_c / sum_c w_c, w_c the
// chunk's sum at the largest reference.  A warp per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_join(const __grid_constant__ Args a) {
    const int block = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Block blk = block_of(a, seq, block, false);
    if (blk.rows == 0 || blk.used == 1) return;
    const int group = a.hq / a.hkv;
    const int64_t unit = (((int64_t)seq * a.hkv + head) * a.blocks + block) * a.chunks;
    for (int row = warp; row < blk.rows; row += kWarps) {
        const float2* st = a.state + unit * 16 + row;
        float m = -INFINITY;
        for (int c = lane; c < blk.used; c += 32) m = fmaxf(m, st[c * 16].x);
        m = tbk::warp_max(m);
        float total = 0.0f, y[kv8::kMaxDim / 32];
#pragma unroll
        for (int i = 0; i < kv8::kMaxDim / 32; ++i) y[i] = 0.0f;
        for (int c = 0; c < blk.used; ++c) {
            const float2 s = st[c * 16];
            const float w = s.x == -INFINITY ? s.y : s.y * exp2f(s.x - m);
            const float* part = a.part + ((unit + c) * 16 + row) * a.d;
            total += w;
#pragma unroll
            for (int i = 0; i < kv8::kMaxDim / 32; ++i)
                if (lane + 32 * i < a.d) y[i] += w * part[lane + 32 * i];
        }
        const bool none = total == 0.0f;
        const int64_t at = (int64_t)block * 16 + row;
        const int64_t tok = blk.s.lo + at / group;
        const int h = head * group + (int)(at % group);
        T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
#pragma unroll
        for (int i = 0; i < kv8::kMaxDim / 32; ++i)
            if (lane + 32 * i < a.d)
                tbk::Elt<T>::store(out + lane + 32 * i, none ? 0.0f : y[i] / total);
        if (a.lse && lane == 0)
            a.lse[tok * a.hq + h] = none ? -INFINITY : m * 0.69314718055994531f + logf(total);
    }
}

int check(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
          bool pointers) {
    int rc = kv8::check_cache(cache, pointers);
    if (rc == TB_OK) rc = kv8::check_batch(batch, pointers);
    if (rc != TB_OK) return rc;
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->n_heads < 1 || t->n_heads > 65535 || t->n_heads % cache->n_kv_heads ||
        t->window < 0 || t->max_rows < 0 || t->max_len < 0)
        return TB_ERR_INVALID_SHAPE;
    const int64_t width = (int64_t)t->n_heads * cache->head_dim;
    if (batch->rows > 1 && pointers && (t->q_stride < width || t->out_stride < width))
        return TB_ERR_INVALID_SHAPE;
    if (pointers && batch->rows && batch->n_seqs && (!t->q || !t->out || t->q == t->out))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

// How a call is cut: blocks of 16 rows per sequence and head, chunks of keys
// per block, scratch.
struct Plan {
    int64_t blocks, chunks;
    size_t part_bytes, state_bytes;
};

Plan plan_of(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
             int sm_count) {
    Plan p;
    const int64_t rows = t->max_rows < batch->rows ? t->max_rows : batch->rows;
    p.blocks = (rows * (t->n_heads / cache->n_kv_heads) + 15) / 16;
    if (p.blocks < 1) p.blocks = 1;
    const int64_t all = p.blocks * cache->n_kv_heads * batch->n_seqs;
    const int64_t slots = 3 * (int64_t)sm_count;
    int64_t keys = t->max_len;
    if (t->window && t->window + rows < keys) keys = t->window + rows;
    const int64_t most = (keys + kLeastChunk - 1) / kLeastChunk;
    p.chunks = all >= slots ? (8 * slots + all - 1) / all : slots / all;
    if (p.chunks > most) p.chunks = most;
    if (p.chunks < 1) p.chunks = 1;
    const size_t units = p.chunks > 1 ? (size_t)(all * p.chunks) : 0;
    p.part_bytes = units * 16 * cache->head_dim * sizeof(float);
    p.state_bytes = units * 16 * sizeof(float2);
    return p;
}

template <typename T, int FORMAT, int DP>
int launch(const Args& a, dim3 grid, cudaStream_t s) {
    constexpr int bytes = smem_bytes<T, DP>();
    TB_CUDA_TRY(cudaFuncSetAttribute(k_attend<T, FORMAT, DP>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    k_attend<T, FORMAT, DP><<<grid, kThreads, bytes, s>>>(a);
    TB_LAUNCH_CHECK("8-bit cache attention kernel");
    return TB_OK;
}

template <typename T, int FORMAT>
int launch_dim(const Args& a, dim3 grid, cudaStream_t s) {
    if (a.d <= 64) return launch<T, FORMAT, 64>(a, grid, s);
    if (a.d <= 128) return launch<T, FORMAT, 128>(a, grid, s);
    return launch<T, FORMAT, 256>(a, grid, s);
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
    const Plan p = plan_of(cache, batch, attention, ds->sm_count);
    *bytes = p.part_bytes + p.state_bytes;
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
    const Plan p = plan_of(cache, batch, t, ds->sm_count);
    if (p.blocks * p.chunks > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    const size_t bytes = p.part_bytes + p.state_bytes;
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
    a.k = static_cast<const uint8_t*>(cache->k);
    a.v = static_cast<const uint8_t*>(cache->v);
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.status = ds->status;
    a.part = static_cast<float*>(t->workspace);
    a.state = reinterpret_cast<float2*>(static_cast<uint8_t*>(t->workspace) + p.part_bytes);
    a.scale = t->scale;
    a.hq = t->n_heads;
    a.hkv = cache->n_kv_heads;
    a.d = cache->head_dim;
    a.window = t->window;
    a.max_rows = t->max_rows;
    a.max_len = t->max_len;
    a.chunks = (int)p.chunks;
    a.blocks = (int)p.blocks;
    a.vec = tbh::aligned16(t->q) && t->q_stride * s % 16 == 0;
    const dim3 grid((unsigned)(p.blocks * p.chunks), (unsigned)a.hkv, (unsigned)batch->n_seqs);
    cudaStream_t st = tbh::stream_of(stream);
    const bool f32 = t->dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    rc = f32 ? (int8 ? launch_dim<float, kv8::kInt8>(a, grid, st)
                     : launch_dim<float, kv8::kE4m3>(a, grid, st))
             : (int8 ? launch_dim<__nv_bfloat16, kv8::kInt8>(a, grid, st)
                     : launch_dim<__nv_bfloat16, kv8::kE4m3>(a, grid, st));
    if (rc != TB_OK || p.chunks == 1) return rc;
    const dim3 joins((unsigned)p.blocks, (unsigned)a.hkv, (unsigned)batch->n_seqs);
    if (f32)
        k_join<float><<<joins, kThreads, 0, st>>>(a);
    else
        k_join<__nv_bfloat16><<<joins, kThreads, 0, st>>>(a);
    TB_LAUNCH_CHECK("8-bit cache attention join kernel");
    return TB_OK;
}
