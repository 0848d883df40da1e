// k_sample_filtered.cu -- one token of each row of logits, after temperature, top-k, top-p
// and min-p.
//
//   w_i = exp((x_i - max x) / temperature) as a whole number of 2^-shift, shift = 62 - the
//   bits of the vocabulary, so that sums fit 64 bits and do not depend on an order;
//   the k first in falling order; of those the ones whose predecessors' weights sum to less
//   than top_p of all; of those the ones with w_i >= min_p; of those, in the order of i, the
//   first whose running sum is above u times the whole.
// What is inside a border in falling order is told by a pair (logit, index): the larger logits,
// and of the equal ones those up to that index.
//
// A row belongs to a cluster of 1 to 8 CTAs, which read it once and keep it in shared memory.
// A border is found from a histogram of 512 bins, 24 for each halving of the weight and one
// for the rest, of counts or of weights (f32, to 2^-15; their sums to 2^-14), that every CTA
// gets of every other: one bin for top-k, for top-p a few that are certain to have it.  For
// top-p what lies above them, and the sum of all, is then summed exactly.  The elements in
// the bins, a few hundred at most, are gathered and ranked by comparing all with all; more of
// them are first thinned by exact histograms of their bits, and equal ones are told apart by a
// search in the order of the index.  That search, by exact sums of CTA, warp, slab and lane,
// makes the draw too.  Where all that is above the border is as few, the last steps are one
// CTA's, on that list; and few of many (top-k up to 192) need no histogram of all: the k-th of
// the threads' largest is a bound that few others are above.
//
// What bounds it: a row's chain of exchanges, its bytes cross HBM once.  256 rows of 128256 f32
// are 2048 CTAs, two an SM by shared memory and registers, so 7 rounds of them:
//   first largest 61 us; no filter 119; the 50 first 104 (138 by the histogram of all, whose
//   atomics are 30), and 0.9 of those 109; min_p 87; the 1000 first 200; 0.9 of all 322, of
//   which the exact sums in double and their search are half; 20 us are the bytes alone.
//   1 row of 32000: first largest 4.2 us, no filter 7.5, the 50 first 10, 0.9 of all 17.5.
// Histograms that each CTA pulled from the others took 15000 to 54000 clocks where they read the
// same bins at once: they are pushed.  Radix passes over the bits with exact sums: 1553 us.
#include <float.h>
#include <math.h>

#include <atomic>

#include "tb_device.cuh"
#include "tb_internal.h"

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMostCtas = 8;
constexpr int kBins = kThreads, kPerHalving = 24;  // bins; the last is for the rest
constexpr int kMostSlabs = 23;  // of 8 KB, in shared memory
constexpr int kFew = kThreads / 2;  // elements that are ranked by comparing all with all
constexpr int64_t kMostVocab = (int64_t)kMostCtas * kMostSlabs * kThreads * 4;  // of f32

struct Args {
    const void* logits;
    int64_t stride;
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    const double* uniforms;
    int32_t* out;
    int vocab, shift, part;  // part: elements a CTA, whole slabs
    int ctas;                // of a cluster
    bool vec;                // rows start on 16 bytes
};

// Bits that compare like the logit (-0 is 0), for numbers.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A row's weights: 2^y, y = (x - top) log2 e / temperature, as 2^(j / 16) 2^f, the first from
// a table (16 doubles, two banks each, so a warp's lookups do not conflict), the second from
// the exponential's series in f ln 2, |f ln 2| < 0.0217, whose first term left out,
// (f ln 2)^7 / 5040, is below 2^-51.
struct Weights {
    float part, part_top, per;  // fall: (part_top - part x) per
    double top, scale;          // y = (x - top) scale
    const double* table;
    int shift;
    // (a temperature above 1 takes half of each logit, whose difference is within f32; one
    // below f32's normal numbers, whose reciprocal is not, does not come here)
    __device__ Weights(float top_, float t, const double* table, int shift)
        : part(t > 1.0f ? 0.5f : 1.0f), part_top(top_ * part), top(top_),
          scale(1.4426950408889634074 / (double)t), table(table), shift(shift) {
        per = (float)(scale / part);
    }
    // How far a logit lies below the top, in halvings of its weight; NaN stays NaN.
    __device__ __forceinline__ float fall(float x) const {
        return __fmul_rn(fmaf(-part, x, part_top), per);
    }
    __device__ __forceinline__ float logit_at(float y) const { return (part_top - y / per) / part; }
    // (no product here that the compiler may or may not fuse with a sum, or a weight could come
    // out a unit more in one place than in another: what is summed in one pass is searched by the
    // sums of a later one)
    __device__ __forceinline__ u64 operator()(float x) const {
        if (!(fall(x) < 64.0f)) return 0;
        constexpr double kLn2 = 0.69314718055994530942;
        constexpr double c2 = kLn2 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4,
                         c5 = c4 * kLn2 / 5, c6 = c5 * kLn2 / 6;
        const double magic = 0x1.8p48;  // a unit of 2^-4
        const double d = (double)x - top, z = fma(d, scale, magic), f = fma(d, scale, magic - z);
        const int n = __double2loint(z);
        double p = fma(f, c6, c5);
        p = fma(f, p, c4);
        p = fma(f, p, c3);
        p = fma(f, p, c2);
        p = fma(f, p, kLn2);
        p = fma(f, p, 1.0);
        const double t = table[n & 15];
        const double unit = __hiloint2double(
            __double2hiint(t) + ((n >> 4) + shift) * (1 << 20), __double2loint(t));
        // a whole number below 2^52 is the low bits of 2^52 more
        return (u64)__double_as_longlong(fma(p, unit, 0x1p52)) - 0x4330000000000000ull;
    }
};

// Whether a logit's weight is min_p or more.
__device__ __forceinline__ bool reaches(float x, double top, double t, double min_p) {
    return exp(((double)x - top) / t) >= min_p;
}

struct Border {
    float x;
    int index;  // the last inside of the logits that are x
    __device__ __forceinline__ bool inside(float v, int i) const {
        return v > x || (v == x && i <= index);
    }
};

// floor(a b / 2^s), and whether anything was cut off.
__device__ __forceinline__ u64 scaled(u64 a, u64 b, int s, bool& cut) {
    const u64 hi = __umul64hi(a, b), lo = a * b;
    cut = lo << (64 - s) != 0;
    return hi << (64 - s) | lo >> s;
}

struct Member {
    float x;
    int index;
    u64 measure;
};

struct alignas(16) Shared {
    union {
        uint32_t bins[kBins];
        u64 exact[kBins];
        Member members[kFew];
    };
    u64 pushed[kMostCtas][kBins];  // of every CTA
    u64 slots[2][kMostCtas][4];    // by turns: what each CTA says
    u64 warps[4][kWarps];
    u64 ranks[kMostCtas], kept[kWarps];  // a search's sums, of the CTAs and of this one's warps
    double table[16];
    double uniform;  // the row's settings, the first CTA's words to all
    float temperature, min_p, top_p;  // (told as pairs)
    int top_k;
    int bin[2];
    u64 before, in_bin;
    float x;
    int index;
    uint32_t listed;
    int over;  // the list is longer than it may be
};

// (lanes may come from different branches: not the aligned form)
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t peer(const void* mine, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(at)
                 : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    return at;
}
__device__ __forceinline__ void store_to(uint32_t at, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void store_to(uint32_t at, u64 v, u64 w) {
    asm volatile("st.shared::cluster.v2.u64 [%0], {%1, %2};" ::"r"(at), "l"(v), "l"(w) : "memory");
}
__device__ __forceinline__ uint32_t add_to(uint32_t at, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
    return old;
}
// BYTES of a setting to shared memory, some time until cp.async.wait_all.
template <int BYTES>
__device__ __forceinline__ void fetch_to(void* smem, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(smem)),
                 "l"(from), "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ u64 warp_scan(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(tbk::kFull, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += up;
    }
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(tbk::kFull, v, o);
    return v;
}

// A CTA's part of a row, elements [lo, lo + part) and NaN where the row has ended: in shared
// memory; a warp has `slabs` x 32 pieces of V neighbouring elements each, one after the other.
template <typename T>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    const Args& a;
    Shared& sh;
    uint4* held;
    int rank, lo, slabs, turn = 0;

    __device__ Row(const Args& a, Shared& sh, uint4* held, int rank)
        : a(a), sh(sh), held(held), rank(rank), lo(rank * a.part),
          slabs(a.part / (kThreads * V)) {}

    __device__ __forceinline__ int place(int slab) const {
        return ((int)(threadIdx.x >> 5) * slabs + slab) * 32 + (threadIdx.x & 31);
    }
    __device__ __forceinline__ int index(int slab) const { return lo + place(slab) * V; }
    __device__ __forceinline__ uint4 fetch(const T* row, int slab) const {
        const int i = index(slab);
        if (a.vec && i + V <= a.vocab) return __ldcs(reinterpret_cast<const uint4*>(row + i));
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (V == 4) {
                w[j] = i + j < a.vocab ? reinterpret_cast<const uint32_t*>(row)[i + j] : ~0u;
            } else {
                const uint16_t* u = reinterpret_cast<const uint16_t*>(row) + i + 2 * j;
                const int left = a.vocab - i - 2 * j;
                w[j] = (left > 0 ? u[0] : 0xffffu) | (left > 1 ? (uint32_t)u[1] : 0xffffu) << 16;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ static void widen(const uint4& raw, float (&v)[V]) {
        tbk::Elt<T>::template widen<V>(raw, v);
    }
    // The row's part to shared memory, and the largest of the thread's elements.
    __device__ __forceinline__ float load(const T* row) {
        constexpr int kAhead = 8;  // pieces asked for at once
        float top = -INFINITY;
        for (int j0 = 0; j0 < slabs; j0 += kAhead) {
            uint4 raw[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (j0 + j < slabs) raw[j] = fetch(row, j0 + j);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (j0 + j >= slabs) break;
                held[place(j0 + j)] = raw[j];
                float v[V];
                widen(raw[j], v);
#pragma unroll
                for (int e = 0; e < V; ++e) top = fmaxf(top, v[e]);
            }
        }
        return top;
    }
    __device__ __forceinline__ void piece(int slab, float (&v)[V]) const {
        widen(held[place(slab)], v);
    }
    // f(logit, index) of each of the thread's elements.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
        for (int j = 0; j < slabs; ++j) {
            float v[V];
            piece(j, v);
#pragma unroll
            for (int e = 0; e < V; ++e) f(v[e], index(j) + e);
        }
    }

    // Sums over the block of v[0 .. SUMS), and maxima of the rest (32 bits), to every CTA:
    // afterwards sh.slots[the turn returned][rank], and the warps' in sh.warps.
    template <int N, int SUMS>
    __device__ __forceinline__ int tell(u64 (&v)[4]) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = turn;
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const u64 s =
                i < SUMS ? warp_sum(v[i]) : __reduce_max_sync(tbk::kFull, (uint32_t)v[i]);
            if (lane == 0) sh.warps[i][warp] = s;
        }
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                u64 s = lane < kWarps ? sh.warps[i][lane] : 0;
                s = i < SUMS ? warp_sum(s) : __reduce_max_sync(tbk::kFull, (uint32_t)s);
                if (lane < a.ctas) store_to(peer(&sh.slots[t][rank][i], lane), s);
            }
        }
        cluster_sync();
        return t;
    }
    // What the CTAs said in turn t, added up or the largest.
    template <int N, int SUMS>
    __device__ __forceinline__ int all(u64 (&v)[4]) {
        const int t = tell<N, SUMS>(v);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = sh.slots[t][0][i];
            for (int c = 1; c < a.ctas; ++c)
                v[i] = i < SUMS ? v[i] + sh.slots[t][c][i] : max(v[i], sh.slots[t][c][i]);
        }
        return t;
    }
    // The sums for locate of what was told as value i of turn t.
    __device__ __forceinline__ void sums_of(int t, int i) {
        if ((int)threadIdx.x < a.ctas) sh.ranks[threadIdx.x] = sh.slots[t][threadIdx.x][i];
        if (threadIdx.x < kWarps) sh.kept[threadIdx.x] = sh.warps[i][threadIdx.x];
        __syncthreads();
    }
    // The index of the element where the running sum of f(logit, index), in the order of the
    // index, first is above target, which is below the sum of all; sh.ranks and sh.kept are
    // its sums.  One lane returns it, all others -1.
    template <typename F>
    __device__ __forceinline__ int locate(u64 target, F f) {
        const int warp = threadIdx.x >> 5;
        for (int c = 0; c < rank; ++c) {
            if (target < sh.ranks[c]) return -1;
            target -= sh.ranks[c];
        }
        if (target >= sh.ranks[rank]) return -1;
        for (int w = 0; w < warp; ++w) {
            if (target < sh.kept[w]) return -1;
            target -= sh.kept[w];
        }
        if (target >= sh.kept[warp]) return -1;
        for (int j = 0; j < slabs; ++j) {
            float x[V];
            piece(j, x);
            u64 each[V], s = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) s += each[e] = f(x[e], index(j) + e);
            const u64 run = warp_scan(s), all = __shfl_sync(tbk::kFull, run, 31);
            if (target >= all) {
                target -= all;
                continue;
            }
            if (target < run - s || target >= run) return -1;
            u64 sum = run - s;
            int at = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sum += each[e];
                at += sum <= target;
            }
            return index(j) + at;
        }
        return -1;
    }

    // Bin threadIdx.x's sum over the cluster, of get(bin) in each CTA.
    template <typename F>
    __device__ __forceinline__ u64 push(F get) {
        constexpr int kPairs = kBins / 2;
        const int b = threadIdx.x % kPairs * 2;
        const u64 v = get(b), w = get(b + 1);
        for (int c = threadIdx.x / kPairs; c < a.ctas; c += kThreads / kPairs)
            store_to(peer(&sh.pushed[rank][b], c), v, w);
        cluster_sync();
        u64 h = 0;
        for (int c = 0; c < a.ctas; ++c) h += sh.pushed[c][threadIdx.x];
        return h;
    }
    // The sum of h over the bins before this thread's, and over all of them.
    __device__ __forceinline__ u64 scan(u64 h, u64& whole) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const u64 run = warp_scan(h);
        if (lane == 31) sh.warps[0][warp] = run;
        __syncthreads();
        u64 before = 0;
        whole = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sh.warps[0][w];
            whole += sh.warps[0][w];
        }
        return before + run - h;
    }
    // The bins (none: the last) where the running sum reaches each of two limits, the sum
    // before the first of them and its own; h: this thread's bin, `before` it.
    __device__ __forceinline__ void reach(u64 h, u64 before, u64 limit0, u64 limit1, int& b0,
                                          int& b1) {
        const int b = threadIdx.x;
        if ((before < limit0 && before + h >= limit0) || (b == kBins - 1 && before + h < limit0)) {
            sh.bin[0] = b;
            sh.before = before;
            sh.in_bin = h;
        }
        if ((before < limit1 && before + h >= limit1) || (b == kBins - 1 && before + h < limit1))
            sh.bin[1] = b;
        __syncthreads();
        b0 = sh.bin[0];
        b1 = sh.bin[1];
    }

    // The members' list, sorted: what of `measure` comes before the thread's member, two
    // threads each.  FALLING: larger logits and equal ones of lower index, else lower indices.
    template <bool FALLING>
    __device__ __forceinline__ u64 sum_before(int n, const Member& mine) const {
        u64 sum = 0;
#pragma unroll 4
        for (int i = threadIdx.x & 1; i < n; i += 2) {
            const Member o = sh.members[i];
            const bool earlier = FALLING ? o.x > mine.x || (o.x == mine.x && o.index < mine.index)
                                         : o.index < mine.index;
            if (earlier) sum += o.measure;
        }
        return sum + __shfl_xor_sync(tbk::kFull, sum, 1);
    }
    __device__ __forceinline__ Member member_of(int n) const {
        const int m = threadIdx.x >> 1;
        return m < n ? sh.members[m] : Member{-INFINITY, INT32_MAX, 0};
    }
    __device__ __forceinline__ u64 block_sum(u64 v) {
        v = warp_sum(v);
        if ((threadIdx.x & 31) == 0) sh.warps[0][threadIdx.x >> 5] = v;
        __syncthreads();
        u64 s = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += sh.warps[0][w];
        __syncthreads();
        return s;
    }

    // What top-p leaves of a sum of weights: whose predecessors' are below it.
    __device__ __forceinline__ static u64 share(u64 sum, float p) {
        bool cut;
        const u64 q = p > 0.0f ? __double2ull_rd((double)p * 0x1p63) : 0ull;
        const u64 limit = scaled(sum, q, 63, cut);
        return max(limit + cut, 1ull);
    }
    __device__ __forceinline__ static u64 target_of(u64 sum, double u) {
        const u64 q = u > 0.0 ? min(__double2ull_rd(u * 0x1p53), (1ull << 53) - 1) : 0ull;
        bool cut;
        return scaled(sum, q, 53, cut);
    }

    // What a search for a border came to.
    enum Found { kBorder, kSums, kDrawn };
    struct Setting {
        int32_t* out;
        float most;  // the thread's largest logit
    };

    // The draw from the list, n members: the k first of them, then top-p (whose limit is
    // p_limit, or, 0, p's share of those k), then min_p.
    __device__ __forceinline__ void draw_few(const Weights& w, int n, u64 k, u64 p_limit,
                                             const Setting& set) {
        Member mine = member_of(n);
        const bool writes = (threadIdx.x & 1) == 0 && (int)(threadIdx.x >> 1) < n;
        const u64 weight = w(mine.x);
        auto hold = [&](bool kept) {  // the list's measures, of the members that are kept
            mine.measure = kept ? weight : 0;
            __syncthreads();
            if (writes) sh.members[threadIdx.x >> 1].measure = mine.measure;
            __syncthreads();
        };
        // (members come with a measure of 1; every lane takes part in the sums)
        u64 sum = sum_before<true>(n, mine);
        hold(mine.measure && sum < k);
        if (sh.top_p < 1.0f) {
            const u64 limit =
                p_limit ? p_limit : share(block_sum(writes ? mine.measure : 0), sh.top_p);
            sum = sum_before<true>(n, mine);
            hold(mine.measure && sum < limit);
        }
        if (sh.min_p > 0.0f)
            hold(mine.measure &&
                 reaches(mine.x, w.top, (double)sh.temperature, (double)sh.min_p));
        const u64 target = target_of(block_sum(writes ? mine.measure : 0), sh.uniform);
        const u64 before = sum_before<false>(n, mine);
        if (writes && before <= target && target < before + mine.measure) *set.out = mine.index;
    }

    // in: to the last element of those inside it, in falling order, whose predecessors sum to
    // less than a limit: of counts, limit; of weights, p times the sum of all.  kSums: and
    // sh.ranks and sh.kept are the weights' sums inside it.  kDrawn: the row is done.
    template <bool BY_WEIGHT>
    __device__ __forceinline__ Found border(const Weights& w, Border& in, u64 limit,
                                            const Setting& set) {
        const int warp = threadIdx.x >> 5;
        // the nearest of 24 bins a halving: it does not fall where the logit falls
        constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23, a unit of 1
        constexpr float kMost = (kBins - 1) / (float)kPerHalving;
        auto bin_of = [&](float y) {
            return __float_as_int(fmaf(fminf(y, kMost), (float)kPerHalving, kMagic)) -
                   __float_as_int(kMagic);
        };
        sh.bins[threadIdx.x] = 0;
        __syncthreads();
        if constexpr (!BY_WEIGHT) {
            // The n-th of the threads' largest is not above the n-th of all, and little below
            // it where threads are many: what is from its bin on is listed at once, if it fits.
            if (limit <= kFew * 3 / 4 && 2 * (int)limit <= min(kThreads * a.ctas, a.vocab / V)) {
                if (set.most > in.x) atomicAdd(&sh.bins[bin_of(w.fall(set.most))], 1u);
                __syncthreads();
                u64 n, h = push([&](int b) -> u64 { return sh.bins[b]; });
                const u64 before = scan(h, n);
                int b0, b1;
                reach(h, before, limit, limit, b0, b1);
                if (n >= limit && b0 < kBins - 1) {
                    // (any logit does that n of the largest are not below: the bin's lower end)
                    const float from = fmaxf(w.logit_at((b0 + 0.51f) / kPerHalving), -FLT_MAX);
                    u64 v[4] = {0, 0, 0, 0};
                    each([&](float x, int i) {
                        if (!(x >= from)) return;
                        ++v[0];
                        if (*(volatile int*)&sh.over) return;
                        const uint32_t at = add_to(peer(&sh.listed, 0), 1);
                        if (at >= kFew) {
                            sh.over = 1;
                            return;
                        }
                        store_to(peer(sh.members + at, 0),
                                 (u64)(uint32_t)i << 32 | __float_as_uint(x), 1ull);
                    });
                    all<1, 1>(v);
                    if (v[0] <= kFew) {
                        if (rank == 0)
                            draw_few(w, (int)v[0], limit, 0, set);
                        return kDrawn;
                    }
                    if (threadIdx.x == 0) sh.listed = 0;
                } else {
                    cluster_sync();  // the pushed bins have been read
                }
                sh.bins[threadIdx.x] = 0;
                __syncthreads();
            }
        }
        uint32_t rest = 0;  // the last bin's: many rows have most of their elements there
        each([&](float x, int i) {
            if (!in.inside(x, i)) return;
            const float y = w.fall(x);
            const int b = bin_of(y);
            uint32_t m = 1;
            if constexpr (BY_WEIGHT) {
                // of the bin's middle (less than 2^-15 of it is nothing), as a whole number
                float part;
                asm("ex2.approx.ftz.f32 %0, %1;"
                    : "=f"(part)
                    : "f"(fmaf((float)b, 1.0f / kPerHalving, -y)));
                m = __float_as_uint(fmaf(part, 32768.0f, 8388608.0f)) - 0x4b000000u;
            }
            if (b == kBins - 1)
                rest += m;
            else
                atomicAdd(&sh.bins[b], m);
        });
        rest = __reduce_add_sync(tbk::kFull, rest);
        if ((threadIdx.x & 31) == 0 && rest) atomicAdd(&sh.bins[kBins - 1], rest);
        __syncthreads();
        // masses in units of 2^-30 of the largest weight
        u64 h = push([&](int b) -> u64 {
            return BY_WEIGHT
                       ? __float2ull_rn((float)sh.bins[b] * exp2f(15.0f - b * (1.0f / kPerHalving)))
                       : sh.bins[b];
        });
        u64 whole, v[4] = {0, 0, 0, 0};
        u64 before = scan(h, whole);
        int b0, b1, t = 0;
        bool few;  // all that is above and in the bins
        if constexpr (BY_WEIGHT) {
            const double mass = fmax((double)sh.top_p, 0.0) * (double)whole;
            reach(h, before, max((u64)(mass * (1 - 0x1p-13)), 1ull),
                  (u64)(mass * (1 + 0x1p-13)) + 1, b0, b1);
            // exact: the sum of all, of what is above the bins, and how many there are
            each([&](float x, int i) {
                if (!in.inside(x, i)) return;
                const int b = bin_of(w.fall(x));
                const u64 m = w(x);
                v[0] += m;
                if (b <= b1) {
                    if (b < b0) v[1] += m;
                    v[2] += b < b0 ? 1ull << 32 : 1ull;
                }
            });
            t = all<3, 3>(v);
            const u64 above = v[2] >> 32;
            v[2] &= 0xffffffffu;
            few = above + v[2] <= kFew;
            limit = share(v[0], sh.top_p);
            if (few)
                v[2] += above;
            else
                limit -= v[1];
        } else {
            if (whole < limit) {  // everything is inside
                cluster_sync();   // the pushed bins have been read
                return kBorder;
            }
            reach(h, before, limit, limit, b0, b1);
            few = sh.before + sh.in_bin <= kFew;
            v[2] = sh.in_bin + (few ? sh.before : 0);
            if (!few) limit -= sh.before;
        }
        // members: the elements inside `in` of those bins (or those above too, if few), with
        // keys [k_lo, k_hi]
        uint32_t k_lo = 0, k_hi = ~0u;
        const int b_from = few ? 0 : b0;
        auto member = [&](float x, int i) {
            if (!in.inside(x, i)) return false;
            const int b = bin_of(w.fall(x));
            return b >= b_from && b <= b1 && key_of(x) >= k_lo && key_of(x) <= k_hi;
        };
        const bool thinned = v[2] > kFew;
        while (v[2] > kFew) {
            u64 ends[4] = {0, 0, 0, 0};
            each([&](float x, int i) {
                if (!member(x, i)) return;
                const uint32_t k = key_of(x);
                ends[0] = max(ends[0], (u64)k);
                ends[1] = max(ends[1], (u64)~k);
            });
            all<2, 0>(ends);
            k_hi = (uint32_t)ends[0];
            k_lo = ~(uint32_t)ends[1];
            if (k_lo == k_hi) {
                // equal logits: the n first of them
                const float x = logit_of(k_hi);
                const u64 unit = BY_WEIGHT ? w(x) : 1ull;
                const u64 n = unit ? (limit + unit - 1) / unit : 1ull;
                if (n >= v[2]) {
                    if (x != in.x) in = {x, INT32_MAX};
                    return kBorder;
                }
                auto tied = [&](float y, int i) { return (u64)(y == x && in.inside(y, i)); };
                u64 c[4] = {0, 0, 0, 0};
                each([&](float y, int i) { c[0] += tied(y, i); });
                sums_of(tell<1, 1>(c), 0);
                c[0] = (u64)(locate(n - 1, tied) + 1);
                all<1, 0>(c);
                in = {x, (int)c[0] - 1};
                return kBorder;
            }
            const int s = max(0, 23 - __clz(k_hi - k_lo));  // the span >> s is below 512
            sh.exact[threadIdx.x] = 0;
            __syncthreads();
            each([&](float x, int i) {
                if (member(x, i))
                    atomicAdd(&sh.exact[(k_hi - key_of(x)) >> s], BY_WEIGHT ? w(x) : 1ull);
            });
            __syncthreads();
            h = push([&](int b) { return sh.exact[b]; });
            before = scan(h, whole);
            int b;
            reach(h, before, limit, limit, b, b);
            limit -= sh.before;
            const uint32_t high = k_hi - ((uint32_t)b << s);
            k_lo = max(high - ((1u << s) - 1), k_lo);
            k_hi = high;
            u64 c[4] = {0, 0, 0, 0};
            each([&](float x, int i) { c[0] += member(x, i); });
            all<1, 1>(c);
            v[2] = c[0];
        }
        // the list: every CTA's, or, where it has all that is left, the first one's
        const int n = (int)v[2], to_ctas = few ? 1 : a.ctas;
        each([&](float x, int i) {
            if (!member(x, i)) return;
            const u64 m = BY_WEIGHT && !few ? w(x) : 1ull;
            Member* to = sh.members + add_to(peer(&sh.listed, 0), 1);
            for (int c = 0; c < to_ctas; ++c)
                store_to(peer(to, c), (u64)(uint32_t)i << 32 | __float_as_uint(x), m);
        });
        cluster_sync();
        if (few) {
            if (rank == 0)
                draw_few(w, n, BY_WEIGHT ? (u64)kFew : limit, BY_WEIGHT ? limit : 0, set);
            return kDrawn;
        }
        if (threadIdx.x == 0) sh.listed = 0;
        Member mine = member_of(n);
        const u64 sum = sum_before<true>(n, mine);
        if (sum < limit && sum + mine.measure >= limit) {
            sh.x = mine.x;
            sh.index = mine.index;
        }
        if constexpr (BY_WEIGHT) {
            // the sums inside: those above the bins, and the members kept, by CTA and warp
            if (thinned) {
                __syncthreads();
                in = {sh.x, sh.index};
                return kBorder;
            }
            __syncthreads();
            if (threadIdx.x % 2 == 0 && mine.measure && sum >= limit)
                sh.members[threadIdx.x >> 1].measure = 0;
            const float x = sh.x;
            const int index = sh.index;
            __syncthreads();
            const int lane = threadIdx.x & 31, per_warp = a.part / kWarps;
            u64 of_rank = 0, of_warp = 0;
            for (int i = lane; i < n; i += 32) {
                const Member m = sh.members[i];
                const int c = m.index / a.part, at = (m.index - c * a.part) / per_warp;
                if (c == warp) of_rank += m.measure;
                if (c == rank && at == warp) of_warp += m.measure;
            }
            of_rank = warp_sum(of_rank);
            of_warp = warp_sum(of_warp);
            if (lane == 0) {
                if (warp < a.ctas) sh.ranks[warp] = of_rank + sh.slots[t][warp][1];
                sh.kept[warp] = of_warp + sh.warps[1][warp];
            }
            __syncthreads();
            in = {x, index};
            return kSums;
        } else {
            __syncthreads();
            in = {sh.x, sh.index};
            return kBorder;
        }
    }
};

// The least logit whose weight is min_p or more, 0 < min_p <= 1, by a whole warp: 32 keys at a
// time, first those around where the logarithm says, then evenly between the nearest known.
__device__ __forceinline__ float least_of(double min_p, float top, double t) {
    const int lane = threadIdx.x & 31;
    uint32_t lo = key_of(-INFINITY), hi = key_of(top);  // below it, and not
    const float guess = (float)((double)top + log(min_p) * t);
    uint32_t from = max(key_of(guess == guess ? guess : top), lo + 16) - 16, step = 1;
    while (hi - lo > 1) {  // a round leaves a 33rd
        const uint32_t key = from + lane * step;
        bool reached = key >= hi;
        if (key > lo && key < hi) reached = reaches(logit_of(key), (double)top, t, min_p);
        const uint32_t yes = __ballot_sync(tbk::kFull, reached);
        const int first = yes ? __ffs(yes) - 1 : 32;
        if (first < 32) hi = min(hi, from + first * step);
        if (first > 0) lo = max(lo, from + (first - 1) * step);
        step = max((hi - lo) / 33, 1u);
        from = lo + step;
    }
    return logit_of(hi);
}

// The settings of row `at`.  One thread of a cluster reads them, once: its CTAs wait for one another
// on every branch that they decide, and a program that writes them during the call (from a stream
// that nothing orders) gets some draw, not CTAs that wait for ever on different branches.
__device__ __forceinline__ void fetch_settings(const Args& a, Shared& sh, int64_t at) {
    fetch_to<8>(&sh.uniform, a.uniforms + at);
    if (a.temperature)
        fetch_to<4>(&sh.temperature, a.temperature + at);
    else
        sh.temperature = 1.0f;
    if (a.min_p)
        fetch_to<4>(&sh.min_p, a.min_p + at);
    else
        sh.min_p = 0.0f;
    if (a.top_p)
        fetch_to<4>(&sh.top_p, a.top_p + at);
    else
        sh.top_p = 1.0f;
    if (a.top_k)
        fetch_to<4>(&sh.top_k, a.top_k + at);
    else
        sh.top_k = 0;
}
// They to the cluster's other CTAs, by that thread; the next cluster_sync makes them seen.
__device__ __forceinline__ void tell_settings(const Args& a, Shared& sh) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    const u64 u = (u64)__double_as_longlong(sh.uniform);
    const u64 v = (u64)__float_as_uint(sh.min_p) << 32 | __float_as_uint(sh.temperature);
    const u64 w = (u64)(uint32_t)sh.top_k << 32 | __float_as_uint(sh.top_p);
    for (int c = 1; c < a.ctas; ++c) {
        store_to(peer(&sh.uniform, c), u);
        store_to(peer(&sh.temperature, c), v);
        store_to(peer(&sh.top_p, c), w);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const Args a) {
    using R = Row<T>;
    extern __shared__ uint4 held[];
    __shared__ Shared sh;
    if (threadIdx.x == 0) sh.listed = sh.over = 0;
    cluster_arrive();
    R row(a, sh, held, blockIdx.x % a.ctas);
    const int64_t at = blockIdx.x / a.ctas;
    const bool tells = row.rank == 0 && threadIdx.x == 0;
    if (tells) fetch_settings(a, sh, at);
    float mine_top = row.load(static_cast<const T*>(a.logits) + at * a.stride);
    u64 v[4] = {key_of(mine_top), 0, 0, 0};
    if (threadIdx.x < 16) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 16);

    cluster_wait();  // every CTA is there to be written to
    if (tells) tell_settings(a, sh);
    // the largest logit, and the first of the largest
    row.template all<1, 0>(v);
    const float t = sh.temperature;
    const int k = sh.top_k;
    float top = logit_of((uint32_t)v[0]);
    if (top == -INFINITY) {
        if (row.rank == 0 && threadIdx.x == 0) a.out[at] = 0;
        return;
    }
    if (!(t >= 0x1p-126f) || sh.min_p > 1.0f) {
        v[0] = 0;
        row.each([&](float x, int i) {
            if (x == top) v[0] = max(v[0], (u64)~(uint32_t)i);
        });
        row.template all<1, 0>(v);
        if (row.rank == 0 && threadIdx.x == 0) a.out[at] = (int32_t)~(uint32_t)v[0];
        return;
    }
    if (top == INFINITY) {
        // alike, and the others without weight: 0 and -infinity
        for (int j = 0; j < row.slabs; ++j) {
            float x[R::V];
            row.piece(j, x);
            T* to = reinterpret_cast<T*>(held + row.place(j));
#pragma unroll
            for (int e = 0; e < R::V; ++e)
                tbk::Elt<T>::store(to + e, x[e] == top ? 0.0f : -INFINITY);
        }
        top = 0.0f;
        mine_top = mine_top == INFINITY ? 0.0f : -INFINITY;
    }
    const Weights w(top, t, sh.table, a.shift);
    const typename R::Setting set = {a.out + at, mine_top};

    // everything above -infinity at first
    Border in = {-INFINITY, -1};
    auto found = R::kBorder;
    if (k > 0 && k < a.vocab) found = row.template border<false>(w, in, k, set);
    if (found == R::kBorder && sh.top_p < 1.0f) found = row.template border<true>(w, in, 0, set);
    if (found == R::kDrawn) return;
    const float least =
        sh.min_p > 0.0f ? least_of((double)sh.min_p, top, (double)sh.temperature) : -INFINITY;
    if (least > in.x) {
        in = {least, INT32_MAX};
        found = R::kBorder;
    }
    auto weight = [&](float x, int i) { return in.inside(x, i) ? w(x) : 0ull; };
    if (found == R::kBorder) {
        v[0] = 0;
        row.each([&](float x, int i) { v[0] += weight(x, i); });
        row.sums_of(row.template tell<1, 1>(v), 0);
    }
    u64 sum = 0;
    for (int c = 0; c < a.ctas; ++c) sum += sh.ranks[c];
    // the first with a running sum above u * all
    const int drawn = row.locate(R::target_of(sum, sh.uniform), weight);
    if (drawn >= 0) *set.out = drawn;
}

template <typename T>
int run(Args& a, int64_t rows, int sm_count, cudaStream_t s) {
    // as many CTAs a row as hold it in 64 KB each (two an SM), and more while the SMs have
    // room for them and there is something to share.  In us, top-k 50 and 0.9 (0.9 alone):
    //   256 rows of 32000: 64 KB each 45 (106), 32 KB 49 (103), 128 KB 57 (159); 128 rows 23
    //   (83), 26 (70), 23 (83); 512 rows of 128256, 8 CTAs each: 217 (676), 128 KB 208 (814)
    //   1 row of 32000 by 8 CTAs 13.8 (22), by the 2 that hold it 17 (33); 32 rows 18.5 (40), 20
    //   (75); 64 rows by 4, for which there is room, 19 (53), by 2 20.5 (78), by 8 27 (57); 256
    //   rows by 2 45 (106), by 8 86 (164)
    constexpr int kSlab = kThreads * 16 / sizeof(T);
    const int64_t slots = 2ll * sm_count;
    a.ctas = 1;
    while (a.ctas < kMostCtas &&
           ((int64_t)a.ctas * 65536 < a.vocab * (int64_t)sizeof(T) ||
            (rows * a.ctas * 2 <= slots && (int64_t)a.ctas * kSlab * 2 < a.vocab)))
        a.ctas *= 2;
    if (rows * a.ctas > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    a.part = (a.vocab + a.ctas * kSlab - 1) / (a.ctas * kSlab) * kSlab;
    static std::atomic<uint64_t> granted{0};  // a bit per device
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    if (!(granted.load() >> ds->device & 1)) {
        TB_CUDA_TRY(cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kMostSlabs * kThreads * 16));
        granted.fetch_or(1ull << ds->device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * a.ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)a.part * sizeof(T);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_sample<T>, a));
    TB_LAUNCH_CHECK("filtered sampling kernel");
    return TB_OK;
}

}  // namespace

extern "C" int tb_b200_sample(const TbB200Sample* t, void* stream) {
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->rows < 0 || t->rows > INT32_MAX || t->vocab < 1 || t->vocab > kMostVocab ||
        (t->rows > 1 && t->stride < t->vocab))
        return TB_ERR_INVALID_SHAPE;
    if (t->rows == 0) return TB_OK;
    if (!t->logits || !t->uniforms || !t->out) return TB_ERR_INVALID_ARG;
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    const int64_t bytes = t->dtype == TB_DTYPE_F32 ? 4 : 2;
    Args a = {t->logits, t->stride, t->temperature, t->top_p, t->min_p, t->top_k,
              t->uniforms, t->out, (int)t->vocab, 50, 0, 1,
              tbh::aligned16(t->logits) && t->stride * bytes % 16 == 0};
    while ((1ll << (62 - a.shift)) < t->vocab) --a.shift;
    cudaStream_t s = tbh::stream_of(stream);
    return t->dtype == TB_DTYPE_F32 ? run<float>(a, t->rows, ds->sm_count, s)
                                    : run<__nv_bfloat16>(a, t->rows, ds->sm_count, s);
}
