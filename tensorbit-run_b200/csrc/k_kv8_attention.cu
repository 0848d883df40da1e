// k_kv8_attention.cu -- attention of Q rows over the paged 8-bit cache.
//
//   s_j = scale q.k_j,  out = sum_j p_j v_j,  p = softmax(s),  k_j = code * page scale
//
// A block holds 8 or 16 rows of one sequence and k/v head: (query token, head
// of the group) pairs, token-major.  Its keys are split into chunks over CTAs
// when there are few blocks; a second kernel joins the chunks.
//
// Within a CTA each of 4 warps takes every fourth step of 16 keys, which lie in
// one page, through a ring of TMA stages of its own: one lane issues two copies
// a step, and no barrier of the CTA is in the loop.  The codes go from shared
// memory to registers with 16-byte loads and
// are converted there, as the left operands of m16n8k16 instructions, so that 8
// rows fill the other side:
//   S^T = K Q^T: lane (g, t) (g = lane / 4, t = lane % 4) holds keys order(g)
//     and order(g) + 8, 16 consecutive elements of each; the head dimension is
//     summed in the order in which that puts it, Q's registers the same;
//   O^T = V^T P^T: S^T's registers, transposed 8 x 8, are P^T's operands; lane
//     (g, t) holds elements 16 g .. 16 g + 15 (of 128) of keys order(2t),
//     order(2t + 1) and those + 8.
// order() and TMA's swizzle (the 16-byte piece c of key r lies at c ^ (r & 7))
// put the 8 lanes of each 16-byte access into different banks.
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

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;          // keys a warp takes at once
constexpr int kLeastChunk = 256;   // keys below which a chunk is not split further
constexpr float kSlack = 4.0f;     // how far (log2) scores may pass a reference
constexpr float kLift = 11.0f;     // weights are held times 2^11: up to 2^15 in f16
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    CUtensorMap k_map, v_map;  // [n_pages * n_kv_heads][page][d] codes
    kv8::Batch b;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride;
    const float *k_scale, *v_scale;
    unsigned* status;
    float* part;    // [seq, kv head, block, chunk][block_rows][d] partial outputs
    float2* state;  // the same, a row's (reference, sum)
    float scale;
    int hq, hkv, d, window, max_rows, max_len, chunks, blocks, block_rows, vec;
};

// What a block of rows attends, the same in both kernels.
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
    const int at = block * a.block_rows;  // rows * group fits an int
    k.rows = max(0, min(a.block_rows, k.s.n * group - at));
    k.lo = k.end = 0;
    if (k.rows > 0) {
        if (k.s.len > a.max_len || k.s.n > a.max_rows ||
            k.s.len > ((int64_t)a.b.width << a.b.page_shift)) {
            if (flag) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
        } else {
            const int p0 = k.s.first + at / group;
            const int p1 = k.s.first + (at + k.rows - 1) / group;
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

// The key (of 8) that row g of an operand stands for.
__device__ __forceinline__ int order(int n) { return n ^ ((n & 1) << 2); }
// Where the 16-byte piece c of a stage's key lies: DP = 64 has rows of 64 bytes
// and that swizzle, DP = 256 two tiles of 128-byte rows.
template <int DP>
__device__ __forceinline__ int place(int key, int c) {
    if constexpr (DP == 64) return key * 64 + (c ^ (key >> 1 & 3)) * 16;
    return (c >> 3) * kStep * 128 + key * 128 + ((c ^ key) & 7) * 16;
}

// Shapes of a kernel for heads of up to DP elements and blocks of 8 NB rows.
template <typename T, int DP, int NB>
struct Shape {
    static constexpr bool kSplit = sizeof(T) == 4;  // hi + lo operands
    static constexpr int kStages = DP == 64 ? 5 : 3;
    static constexpr int kStageBytes = 2 * kStep * DP;
    static constexpr int kSteps = DP / 16;                // 16-wide steps of the head dimension
    static constexpr int kRows = 8 * NB;
    // Q's operands stay in registers when they are few
    static constexpr bool kQReg = kSteps * 2 * NB * (kSplit ? 2 : 1) <= 32;
    static constexpr int kQBytes = kQReg ? 0 : kSteps * NB * 256 * (kSplit ? 2 : 1);
    static constexpr int kRing = kWarps * kStages * kStageBytes;  // a multiple of 1024
    static constexpr int kPitch = DP + 4;
    static constexpr int kJoin = kWarps * kRows * (kPitch + 3) * 4;
    static constexpr int kBytes = (kRing > kJoin ? kRing : kJoin) + kQBytes + 1024;  // 1024: to align
    // CTAs per SM: what registers (O: DP NB / 4 a lane) and shared memory allow
    static constexpr int kCtas = DP * NB >= 512 ? 2 : DP * NB >= 256 ? (DP == 256 ? 2 : 3) : 4;
};

template <typename T, int FORMAT, int DP, int NB>
__global__ void __launch_bounds__(kThreads, Shape<T, DP, NB>::kCtas)
k_attend(const __grid_constant__ Args a) {
    using H = Shape<T, DP, NB>;
    constexpr bool kSplit = H::kSplit, kQReg = H::kQReg;
    constexpr int kSteps = H::kSteps, kStages = H::kStages, kRows = H::kRows;
    constexpr int kTiles = DP / 16;  // 16-wide output tiles
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[kWarps * kStages];
    // TMA's swizzle goes by the address: tiles start on 1024 bytes
    uint8_t* smem = smem_raw + (-tbk::smem_addr(smem_raw) & 1023u);

    const int c = blockIdx.x % a.chunks, block = blockIdx.x / a.chunks;
    const int head = blockIdx.y, seq = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Block blk = block_of(a, seq, block, threadIdx.x == 0 && c == 0 && head == 0);
    if (blk.rows == 0 || c >= blk.used) return;
    const int group = a.hq / a.hkv;
    const int begin = blk.from + c * blk.size, end = min(begin + blk.size, blk.end);

    // the warp's steps: keys first + 64 n .. + 15
    const int first = begin + warp * kStep;
    const int n_steps = end > first ? (end - first + kWarps * kStep - 1) / (kWarps * kStep) : 0;
    uint8_t* ring = smem + warp * kStages * H::kStageBytes;
    uint64_t* bar = bars + warp * kStages;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kStages; ++i) tbk::mbar_init(bar + i, 1);
        tbk::fence_mbar_init();
    }
    __syncwarp();
    const int32_t* table = a.b.table + seq * a.b.table_stride;
    auto page_of = [&](int n) {  // the page of step n, -1 if it has none
        if (n >= n_steps) return -1;
        const int id = table[(first + n * (kWarps * kStep)) >> a.b.page_shift];
        if (id >= 0 && id < a.b.n_pages) return id;
        atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
        return -1;
    };
    // Lane i has the page of step 32 m + i and its scales, m the batch that is
    // being issued; the next batch's pages are on their way.
    int ids = page_of(lane), ids_next = page_of(32 + lane);
    float ks_issued = 0.0f, vs_issued = 0.0f, ks = 0.0f, vs = 0.0f;
    uint32_t pages_issued, pages = 0;  // which steps of the batch have a page
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
        if ((n & 31) == 0 && n > 0) {
            ids = ids_next;
            load_scales();
            ids_next = page_of(n + 32 + lane);
        }
        const int id = __shfl_sync(tbk::kFull, ids, n & 31);
        if (lane == 0 && id >= 0) {
            uint8_t* dst = ring + stage * H::kStageBytes;
            const int slot = (first + n * (kWarps * kStep)) & ((1 << a.b.page_shift) - 1);
            tbk::mbar_expect_tx(bar + stage, H::kStageBytes);
#pragma unroll
            for (int h = 0; h < (DP + 127) / 128; ++h) {
                kv8::tma_load3(dst + h * kStep * 128, &a.k_map, h * 128, slot, id * a.hkv + head,
                               bar + stage);
                kv8::tma_load3(dst + kStep * DP + h * kStep * 128, &a.v_map, h * 128, slot,
                               id * a.hkv + head, bar + stage);
            }
        }
    };
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) issue(n, n);

    // Q's operands: rows g, g + 8, .. of the block; a row's scores are
    // multiplied with qf, but for the page's scale
    uint32_t qr[kQReg ? kSteps : 1][NB][2], ql[kQReg && kSplit ? kSteps : 1][NB][2];
    uint2* qs = reinterpret_cast<uint2*>(smem + H::kBytes - 1024 - H::kQBytes);
    float qf[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int i = 8 * b + g;
        const bool live = i < blk.rows;
        const int at = block * kRows + i, tok = live ? at / group : 0;
        const int hh = live ? at - tok * group : 0;
        const T* q = static_cast<const T*>(a.q) + (blk.s.lo + tok) * a.q_stride +
                     (int64_t)(head * group + hh) * a.d;
        float top = 0.0f;
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) {
            float x[16];
            kv8::load16(q + 64 * h + 16 * t, live && 64 * h + 16 * t < a.d, a.vec, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        top = fmaxf(top, __shfl_xor_sync(tbk::kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(tbk::kFull, top, 2));
        // 2^e with |q| 2^e in [2^14, 2^15); NaN and infinite rows stay that
        const int e = min(max((int)(__float_as_uint(top) >> 23), 1 + 16), 254);
        const float lift = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23);
        qf[b] = __uint_as_float((uint32_t)(e - 14) << 23) * (a.scale * kLog2e);
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) {
            float x[16];
            kv8::load16(q + 64 * h + 16 * t, live && 64 * h + 16 * t < a.d, a.vec, x);
#pragma unroll
            for (int e16 = 0; e16 < 16; ++e16) x[e16] *= lift;
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // a word of 4 codes
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float u = x[4 * j + kv8::word_element<FORMAT>(r, 0)];
                    const float w = x[4 * j + kv8::word_element<FORMAT>(r, 1)];
                    hi[r] = kv8::pack_f16x2(u, w);
                    const __half2 h2 = *reinterpret_cast<const __half2*>(&hi[r]);
                    lo[r] = kv8::pack_f16x2(u - __low2float(h2), w - __high2float(h2));
                }
                const int s = 4 * h + j;
                if constexpr (kQReg) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        qr[s][b][r] = hi[r];
                        if (kSplit) ql[s][b][r] = lo[r];
                    }
                } else if (warp == 0) {
                    qs[(s * NB + b) * 32 + lane] = make_uint2(hi[0], hi[1]);
                    if (kSplit) qs[((kSteps + s) * NB + b) * 32 + lane] = make_uint2(lo[0], lo[1]);
                }
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
            const int p = blk.s.first + (block * kRows + i) / group;
            see_hi[b][e] = live ? p : INT32_MAX;
            see_lo[b][e] = a.window && live ? max(p - a.window + 1, 0) : 0;
        }

    if constexpr (!kQReg) __syncthreads();

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
            ref[b][e] = vref[b][e] = -INFINITY;
            sum[b][e] = 0.0f;
        }

    const int ka = order(2 * t), kb = order(2 * t + 1), kg = order(g);
    uint32_t phases = 0;  // of each stage's barrier: a page out of range has no copy
    int at_stage = kStages - 1;
    for (int n = 0; n < n_steps; ++n) {
        if ((n & 31) == 0) {
            ks = ks_issued;
            vs = vs_issued;
            pages = pages_issued;
        }
        __syncwarp();  // step n - 1's stage has been read: it is the next to be filled
        issue(n + kStages - 1, at_stage);
        at_stage = at_stage == kStages - 1 ? 0 : at_stage + 1;
        if (!(pages >> (n & 31) & 1)) continue;
        const float k_scale = __shfl_sync(tbk::kFull, ks, n & 31);
        const float v_scale = __shfl_sync(tbk::kFull, vs, n & 31);
        uint8_t* stage = ring + at_stage * H::kStageBytes;
        const uint32_t phase = phases >> at_stage & 1;
        phases ^= 1u << at_stage;
        const bool came = tbk::mbar_wait(bar + at_stage, phase, a.status);
        if (!__all_sync(tbk::kFull, came)) {
            // the copy did not come: the output is invalid and flagged.  No copy
            // may be in flight when the block ends: wait for the others, bounded.
            for (int i = 1; i < kStages; ++i) {
                const int m = n + i, x = (at_stage + i) % kStages;
                const int id = m < n_steps ? table[(first + m * (kWarps * kStep)) >> a.b.page_shift]
                                           : -1;
                if (id >= 0 && id < a.b.n_pages)
                    tbk::mbar_wait(bar + x, phases >> x & 1, a.status);
            }
            break;
        }
        const int key0 = first + n * (kWarps * kStep);
        if (key0 + kStep > blk.s.len) {
            // slots behind the last token may hold anything, NaN codes too: a
            // weight of zero needs a finite value beside it
            for (int i = lane; i < kStep * DP / 16; i += 32)
                if (key0 + i % kStep >= blk.s.len)
                    *reinterpret_cast<uint4*>(stage + kStep * DP +
                                              place<DP>(i % kStep, i / kStep)) =
                        make_uint4(0, 0, 0, 0);
            __syncwarp();
        }

        // S^T: 16 keys by the block's rows, two sums of half the steps each
        float s2[2][NB][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) s2[i][b][e] = 0.0f;
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) {
            const uint4 x =
                *reinterpret_cast<const uint4*>(stage + place<DP>(kg, 4 * h + t));
            const uint4 y =
                *reinterpret_cast<const uint4*>(stage + place<DP>(kg + 8, 4 * h + t));
            const uint32_t wx[4] = {x.x, x.y, x.z, x.w}, wy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a0, a1, a2, a3;
                kv8::word<FORMAT>(wx[j], a0, a2);
                kv8::word<FORMAT>(wy[j], a1, a3);
                const int k = 4 * h + j;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if constexpr (kQReg) {
                        kv8::mma16816(s2[j & 1][b], a0, a1, a2, a3, qr[k][b][0], qr[k][b][1]);
                        if constexpr (kSplit)
                            kv8::mma16816(s2[j & 1][b], a0, a1, a2, a3, ql[k][b][0], ql[k][b][1]);
                    } else {
                        const uint2 q = qs[(k * NB + b) * 32 + lane];
                        kv8::mma16816(s2[j & 1][b], a0, a1, a2, a3, q.x, q.y);
                        if constexpr (kSplit) {
                            const uint2 r = qs[((kSteps + k) * NB + b) * 32 + lane];
                            kv8::mma16816(s2[j & 1][b], a0, a1, a2, a3, r.x, r.y);
                        }
                    }
                }
            }
        }
        // log2 units: s[b][2 i + e] is key key0 + kg + 8 i, row 8 b + 2 t + e; the
        // values' scale as an exponent
        const float lv = (float)((int)(__float_as_uint(v_scale) >> 23) - 127);
        float s[NB][4];
        bool inside = true, over = false;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = qc[b][e] * k_scale;
                s[b][e] = (s2[0][b][e] + s2[1][b][e]) * f;
                s[b][2 + e] = (s2[0][b][2 + e] + s2[1][b][2 + e]) * f;
                inside &= key0 >= see_lo[b][e] && key0 + kStep - 1 <= see_hi[b][e];
            }
        if (!__all_sync(tbk::kFull, inside)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = key0 + kg + 8 * (i >> 1);
                    if (j < see_lo[b][i & 1] || j > see_hi[b][i & 1]) s[b][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float hi = fmaxf(s[b][e], s[b][2 + e]);
                over |= hi > ref[b][e] + kSlack || hi + lv > vref[b][e] + kSlack;
            }
        if (__any_sync(tbk::kFull, over)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float hi = fmaxf(s[b][e], s[b][2 + e]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1)
                        hi = fmaxf(hi, __shfl_xor_sync(tbk::kFull, hi, x));
                    const float m = fmaxf(ref[b][e], ceilf(hi));
                    const float mv = fmaxf(vref[b][e], ceilf(hi) + lv);
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
        // weights: for the sum, and times the values' scale as P^T's operands
        uint32_t ph[NB][2], pl[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float m = ref[b][e] == -INFINITY ? 0.0f : ref[b][e];
                const float mv = (vref[b][e] == -INFINITY ? 0.0f : vref[b][e]) - lv - kLift;
                sum[b][e] += kv8::exp2_fast(s[b][e] - m) + kv8::exp2_fast(s[b][2 + e] - m);
                p[e] = kv8::exp2_fast(s[b][e] - mv);
                p[2 + e] = kv8::exp2_fast(s[b][2 + e] - mv);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t hi = kv8::pack_f16x2(p[2 * i], p[2 * i + 1]);
                ph[b][i] = kv8::transpose8(hi);
                if constexpr (kSplit) {
                    const __half2 h2 = *reinterpret_cast<const __half2*>(&hi);
                    pl[b][i] = kv8::transpose8(kv8::pack_f16x2(p[2 * i] - __low2float(h2),
                                                               p[2 * i + 1] - __high2float(h2)));
                }
            }
        }
        // O^T += V^T P^T: tile rows g and g + 8 are two neighbouring elements
        const uint8_t* values = stage + kStep * DP;
        constexpr int kWide = DP >= 128 ? 16 : 8;  // bytes a lane takes of a key at once
#pragma unroll
        for (int h = 0; h < (DP + 127) / 128; ++h) {
            uint32_t w[4][kWide / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = (i & 1 ? kb : ka) + (i & 2 ? 8 : 0);
                if constexpr (DP >= 128) {
                    const uint4 x =
                        *reinterpret_cast<const uint4*>(values + place<DP>(key, 8 * h + g));
                    w[i][0] = x.x;
                    w[i][1] = x.y;
                    w[i][2] = x.z;
                    w[i][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(
                        values + place<DP>(key, g >> 1) + (g & 1) * 8);
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
                        kv8::mma16816(d, lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1],
                                      ph[b][0], ph[b][1]);
                        if constexpr (kSplit)
                            kv8::mma16816(d, lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1],
                                          pl[b][0], pl[b][1]);
                    }
            }
        }
    }
    __syncthreads();  // the rings are free: the warps' states meet in their place

    // o[h 8 + u][b][2 r + e]: element 128 h + kWide g + 2 u + r of row 8 b + 2 t + e
    constexpr int kWide = DP >= 128 ? 16 : 8;
    float* jo = reinterpret_cast<float*>(smem);
    float* jm = jo + kWarps * kRows * H::kPitch;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float z = sum[b][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(tbk::kFull, z, x);
            const int i = warp * kRows + 8 * b + 2 * t + e;
            float* row = jo + i * H::kPitch;
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
                *reinterpret_cast<float2*>(row + (u / 8) * 128 + kWide * g + 2 * (u % 8)) =
                    make_float2(o[u][b][e], o[u][b][2 + e]);
            if (g == 0) {
                jm[i * 3] = ref[b][e];
                jm[i * 3 + 1] = vref[b][e];
                jm[i * 3 + 2] = z;
            }
        }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool whole = blk.used == 1;
    const int64_t unit =
        (((int64_t)seq * a.hkv + head) * a.blocks + block) * a.chunks + c;
    for (int row = warp; row < blk.rows; row += kWarps) {
        float m = -INFINITY, mv = -INFINITY, total = 0.0f, w[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            m = fmaxf(m, jm[(i * kRows + row) * 3]);
            mv = fmaxf(mv, jm[(i * kRows + row) * 3 + 1]);
        }
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float* st = jm + (i * kRows + row) * 3;
            total += st[0] == -INFINITY ? st[2] : st[2] * exp2f(st[0] - m);
            w[i] = st[1] == -INFINITY ? 0.0f : exp2f(st[1] - mv);
        }
        const bool none = total == 0.0f;
        // O is in units of 2^(mv - lift), the sum of 2^m
        const float per = none ? 0.0f : exp2f(-kLift) / total;
        const float unit_v = none ? 0.0f : exp2f(mv - m);
        const int at = block * kRows + row;
        const int64_t tok = blk.s.lo + at / group;
        const int h = head * group + at % group;
        T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
        float* part = whole ? nullptr : a.part + (unit * kRows + row) * a.d;
        for (int i = lane; i < a.d; i += 32) {
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) y += w[k] * jo[(k * kRows + row) * H::kPitch + i];
            y = none ? 0.0f : y * per * unit_v;
            if (whole)
                tbk::Elt<T>::store(out + i, y);
            else
                part[i] = y;
        }
        if (lane == 0) {
            if (!whole)
                a.state[unit * kRows + row] = make_float2(m, total);
            else if (a.lse)
                a.lse[tok * a.hq + h] = none ? -INFINITY : m * 0.69314718055994531f + logf(total);
        }
    }
}

// Joins the chunks of a row: out = sum_c w_c out_c / sum_c w_c, w_c the chunk's
// sum at the largest reference.  A CTA per row: the weights first, then a warp
// takes every eighth chunk, four loads in flight, a lane four elements of 128.
constexpr int kJoinWarps = 8;
constexpr int kMostChunks = 1024;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) k_join(const __grid_constant__ Args a) {
    __shared__ float w_s[kMostChunks];
    __shared__ float4 part[kJoinWarps][kv8::kMaxDim / 4];
    __shared__ float red[32];
    const int block = blockIdx.x / a.block_rows, row = blockIdx.x % a.block_rows;
    const int head = blockIdx.y, seq = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Block blk = block_of(a, seq, block, false);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= blk.rows || blk.used == 1) return;
    const int group = a.hq / a.hkv;
    const int64_t unit = (((int64_t)seq * a.hkv + head) * a.blocks + block) * a.chunks;
    const float2* st = a.state + unit * a.block_rows + row;
    const float4* parts = reinterpret_cast<const float4*>(a.part) + (unit * a.block_rows + row) * (a.d / 4);
    const int64_t pitch = (int64_t)a.block_rows * (a.d / 4);
    float m = -INFINITY;
    for (int c = threadIdx.x; c < blk.used; c += 32 * kJoinWarps)
        m = fmaxf(m, st[(int64_t)c * a.block_rows].x);
    m = tbk::block_max(m, red);
    float mine = 0.0f;
    for (int c = threadIdx.x; c < blk.used; c += 32 * kJoinWarps) {
        const float2 s = st[(int64_t)c * a.block_rows];
        const float w = s.x == -INFINITY ? s.y : s.y * exp2f(s.x - m);
        w_s[c] = w;
        mine += w;
    }
    const float total = tbk::group_sum(mine, 32 * kJoinWarps, red);  // and w_s is written
#pragma unroll
    for (int h = 0; h < kv8::kMaxDim / 128; ++h) {
        const int i = 32 * h + lane;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < a.d / 4) {
            for (int c0 = warp; c0 < blk.used; c0 += 4 * kJoinWarps) {
                float4 x[4];
                float w[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int c = c0 + u * kJoinWarps;
                    const bool there = c < blk.used;
                    w[u] = there ? w_s[c] : 0.0f;
                    x[u] = there ? __ldcg(parts + c * pitch + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    y.x = fmaf(w[u], x[u].x, y.x);
                    y.y = fmaf(w[u], x[u].y, y.y);
                    y.z = fmaf(w[u], x[u].z, y.z);
                    y.w = fmaf(w[u], x[u].w, y.w);
                }
            }
            part[warp][i] = y;
        }
    }
    __syncthreads();
    const bool none = total == 0.0f;
    const int at = block * a.block_rows + row;
    const int64_t tok = blk.s.lo + at / group;
    const int h = head * group + at % group;
    T* out = static_cast<T*>(a.out) + tok * a.out_stride + (int64_t)h * a.d;
    for (int i = threadIdx.x; i < a.d; i += 32 * kJoinWarps) {
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinWarps; ++k) z += reinterpret_cast<const float*>(part[k])[i];
        tbk::Elt<T>::store(out + i, none ? 0.0f : z / total);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[tok * a.hq + h] = none ? -INFINITY : m * 0.69314718055994531f + logf(total);
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
    // a sequence's (token, head of the group) rows are counted in an int
    if (batch->rows * (t->n_heads / cache->n_kv_heads) > INT32_MAX / 2) return TB_ERR_INVALID_SHAPE;
    const int64_t width = (int64_t)t->n_heads * cache->head_dim;
    if (batch->rows > 1 && pointers && (t->q_stride < width || t->out_stride < width))
        return TB_ERR_INVALID_SHAPE;
    if (pointers && batch->rows && batch->n_seqs && (!t->q || !t->out || t->q == t->out))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

// How a call is cut: blocks of rows per sequence and head, chunks of keys per
// block, scratch.
struct Plan {
    int64_t blocks, chunks;
    int block_rows;
    size_t part_bytes, state_bytes;
};

Plan plan_of(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
             int sm_count) {
    Plan p;
    const int64_t rows = t->max_rows < batch->rows ? t->max_rows : batch->rows;
    const int64_t most_rows = rows * (t->n_heads / cache->n_kv_heads);
    p.block_rows = most_rows <= 8 ? 8 : 16;
    p.blocks = (most_rows + p.block_rows - 1) / p.block_rows;
    if (p.blocks < 1) p.blocks = 1;
    const int64_t all = p.blocks * cache->n_kv_heads * batch->n_seqs;
    const int64_t slots = (p.block_rows == 8 ? 4 : 3) * (int64_t)sm_count;
    int64_t keys = t->max_len;
    if (t->window && t->window + rows < keys) keys = t->window + rows;
    const int64_t most = (keys + kLeastChunk - 1) / kLeastChunk;
    p.chunks = 2 * all > slots ? (8 * slots + all - 1) / all : slots / all;
    if (p.chunks > most) p.chunks = most;
    if (p.chunks > kMostChunks) p.chunks = kMostChunks;
    if (p.chunks < 1) p.chunks = 1;
    const size_t units = p.chunks > 1 ? (size_t)(all * p.chunks) : 0;
    p.part_bytes = units * p.block_rows * cache->head_dim * sizeof(float);
    p.state_bytes = units * p.block_rows * sizeof(float2);
    return p;
}

template <typename T, int FORMAT, int DP, int NB>
int launch(Args& a, const TbB200Kv8* cache, dim3 grid, cudaStream_t s) {
    constexpr int bytes = Shape<T, DP, NB>::kBytes;
    static std::atomic<uint64_t> granted{0};  // a bit per device
    int rc = kv8::once_per_device(granted, [&] {
        return cudaFuncSetAttribute(k_attend<T, FORMAT, DP, NB>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    });
    if (rc == TB_OK) rc = kv8::tile_map(&a.k_map, cache, cache->k, DP < 128 ? DP : 128, kStep);
    if (rc == TB_OK) rc = kv8::tile_map(&a.v_map, cache, cache->v, DP < 128 ? DP : 128, kStep);
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

template <typename T>
int join(const Args& a, dim3 grid, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * kJoinWarps);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_join<T>, a));
    TB_LAUNCH_CHECK("8-bit cache attention join kernel");
    return TB_OK;
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
    if (p.blocks * p.chunks > INT32_MAX || p.blocks * p.block_rows > INT32_MAX) return TB_ERR_INVALID_SHAPE;
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
    a.block_rows = p.block_rows;
    a.vec = tbh::aligned16(t->q) && t->q_stride * s % 16 == 0;
    const dim3 grid((unsigned)(p.blocks * p.chunks), (unsigned)a.hkv, (unsigned)batch->n_seqs);
    cudaStream_t st = tbh::stream_of(stream);
    const bool f32 = t->dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    rc = f32 ? (int8 ? launch_rows<float, kv8::kInt8>(a, cache, grid, st)
                     : launch_rows<float, kv8::kE4m3>(a, cache, grid, st))
             : (int8 ? launch_rows<__nv_bfloat16, kv8::kInt8>(a, cache, grid, st)
                     : launch_rows<__nv_bfloat16, kv8::kE4m3>(a, cache, grid, st));
    if (rc != TB_OK || p.chunks == 1) return rc;
    const dim3 joins((unsigned)(p.blocks * p.block_rows), (unsigned)a.hkv, (unsigned)batch->n_seqs);
    return f32 ? join<float>(a, joins, st) : join<__nv_bfloat16>(a, joins, st);
}
