// Rows of logits over a vocabulary: log probabilities of given tokens with entropies and the best alternatives, and the
// distillation loss against a teacher's best tokens, each with the gradient of the logits.
//
// With y = x / temperature, m the row's largest logit and t_j = (x_j - m) / temperature, everything that a row needs is
//   S = sum exp(t_j),   W = sum exp(t_j) t_j,   log p_j = t_j - log S,   entropy = log S - W / S
// and a handful of single logits.  The exponent is taken after the subtraction, so no large numbers meet in it, whatever
// the temperature; sums run in fp32 per thread and are joined in 64 bits, where the few values per row are finished too.
//
// Bound by HBM (one read of the logits forward, a read and a write backward): a CTA of 256 threads streams a row, or its
// part of a row, with 16-byte loads and a running maximum per thread; rows are split over a cluster of up to 8 CTAs when
// there are few of them, and joined through distributed shared memory: one launch, no workspace, a fixed order of sums.
// Included by lme_cuda.cu after decode_attention.cu.
#include <cuda_fp16.h>

namespace lme {
namespace vr {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int UNROLL = 4;               // vectors of 16 bytes per thread and step
constexpr int MAX_SPLITS = 8;           // CTAs of a cluster
constexpr int MAX_K = LME_VOCAB_MAX_K;  // best tokens, or tokens of a teacher, per row
constexpr int SEGMENTS = 4;             // of a CTA's steps: the maxima that the selection starts from
constexpr int MAX_CANDIDATES = 2048;
constexpr int MAX_MAP = 96 * 1024;      // bytes of the map of listed tokens: a byte per vector of a CTA
constexpr float T_MIN = -150.f;         // 2^-150 is zero here; keeps 0 * (-inf) out of the sums
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;

// ------------------------------------------------------------------ element types
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int N = 8;         // per vector
    static constexpr int KEY_BITS = 16; // of an ordered key that differ between values
    static constexpr uint32_t NEG_INF = 0xff80ff80u;
    static __device__ __forceinline__ float f(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) { unpack8(u, f); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float max_halves(uint32_t w) {
        const float2 v = unpack_bf16x2(w);
        return max_nan(v.x, v.y);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
    static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<__half> {
    static constexpr int N = 8;
    static constexpr int KEY_BITS = 19; // fp16 as fp32 bits: 13 zeros at the end
    static constexpr uint32_t NEG_INF = 0xfc00fc00u;
    static __device__ __forceinline__ float f(__half x) { return __half2float(x); }
    static __device__ __forceinline__ float2 two(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = two(w[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float max_halves(uint32_t w) {
        const float2 v = two(w);
        return max_nan(v.x, v.y);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
    }
    static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<float> {
    static constexpr int N = 4;
    static constexpr int KEY_BITS = 20; // the selection's first bound may be coarse
    static constexpr uint32_t NEG_INF = 0xff800000u;
    static __device__ __forceinline__ float f(float x) { return x; }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x);
        f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z);
        f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ float max_halves(uint32_t w) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float from(float x) { return x; }
};

// ------------------------------------------------------------------ rows and their slices
// Row r starts at x + (r / inner) * ld_outer + (r % inner) * ld_inner: sequences whose last positions are left out are
// read in place.
struct Rows {
    const void* x;
    long long inner, ld_inner, ld_outer;
    int V;
    template <typename T>
    __device__ __forceinline__ const T* row(long long r) const {
        const long long o = r / inner;
        return static_cast<const T*>(x) + o * ld_outer + (r - o * inner) * ld_inner;
    }
};

// The vectors of a row are the 16-byte pieces of memory that it lies in, so rows may start at any element; its first and
// its last vector may be parts, which are read element by element.
template <typename T>
struct Slice {
    static constexpr int N = Elem<T>::N;
    const T* row;
    int V, before;              // before: elements between the first vector's start and the row's
    int nv, begin, end;         // vectors of the row, and those of this CTA
    int full0, full1;           // whole ones among them
    bool head, tail;            // whether this CTA has a part at the start / at the end

    __device__ __forceinline__ Slice(const T* row_, int V_, int rank, int splits) : row(row_), V(V_) {
        before = static_cast<int>((reinterpret_cast<uintptr_t>(row_) & 15) / sizeof(T));
        nv = (before + V + N - 1) / N;
        const int per = (nv + splits - 1) / splits;
        begin = min(nv, rank * per);
        end = min(nv, begin + per);
        const bool ragged = (before + V) % N != 0;
        head = begin == 0 && end > 0 && (before > 0 || (nv == 1 && ragged));
        tail = end == nv && end > begin && nv > 1 && ragged;
        full0 = begin + (head ? 1 : 0);
        full1 = end - (tail ? 1 : 0);
    }
    __device__ __forceinline__ int index(int j, int e) const { return j * N + e - before; }
    __device__ __forceinline__ bool has(int id) const {     // whether token `id` is in this CTA's vectors
        const int j = (id + before) / N;
        return id >= 0 && id < V && j >= begin && j < end;
    }
    __device__ __forceinline__ uint4 load(int j) const {    // a whole vector
        const T* p = row - before + static_cast<long long>(j) * N;
        uint4 r;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
        return r;
    }
    static __device__ __forceinline__ uint4 nothing() {
        constexpr uint32_t w = Elem<T>::NEG_INF;
        return make_uint4(w, w, w, w);
    }
    // a part, minus infinity where the row is not
    __device__ __forceinline__ uint4 load_part(int j) const {
        uint4 r = nothing();
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = index(j, i);
            if (v >= 0 && v < V) e[i] = row[v];
        }
        return r;
    }
    __device__ __forceinline__ bool whole(int j) const { return j >= full0 && j < full1; }
    __device__ __forceinline__ uint4 load_any(int j) const { return whole(j) ? load(j) : load_part(j); }
    __device__ __forceinline__ int steps() const { return (full1 - full0 + THREADS * UNROLL - 1) / (THREADS * UNROLL); }
};

template <typename T, int U>
__device__ __forceinline__ float max_of(const uint4 (&r)[U]) {
    uint32_t w = r[0].x;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        w = Elem<T>::max2(w, r[u].x);
        w = Elem<T>::max2(w, r[u].y);
        w = Elem<T>::max2(w, r[u].z);
        w = Elem<T>::max2(w, r[u].w);
    }
    return Elem<T>::max_halves(w);
}

// ------------------------------------------------------------------ running sums of a thread
// m: largest logit so far, s: sum of 2^t, w: sum of 2^t t with t = (x - m) c.  A NaN reaches all three.
template <bool ENTROPY, bool TWO>
struct Running {
    float m = -INFINITY, s = 0.f, w = 0.f, s1 = 0.f;    // s1: s at temperature one (c1)

    __device__ __forceinline__ void raise(float to, float c, float c1) {
        const float d = m - to;
        const float t = max_nan(d * c, T_MIN);          // (-inf) - (-inf) cannot be: `to` is above m
        const float f = exp2_approx(t);
        if (ENTROPY) w = (w + s * t) * f;
        s *= f;
        if (TWO) s1 *= exp2_approx(max_nan(d * c1, T_MIN));
        m = to;
    }
    template <typename T, int U>
    __device__ __forceinline__ void add(const uint4 (&r)[U], float largest, float c, float c1) {
        constexpr int N = Elem<T>::N;
        if (!(largest <= m)) raise(largest, c, c1);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[N];
            Elem<T>::unpack(r[u], f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float d = f[e] - base;
                const float t = max_nan(d * c, T_MIN);
                const float p = exp2_approx(t);
                s += p;
                if (ENTROPY) w = fmaf(p, t, w);
                if (TWO) s1 += exp2_approx(max_nan(d * c1, T_MIN));
            }
        }
    }
};
// The CTA's sums, relative to its largest logit, in every thread (`red`: 4 * WARPS floats).
struct Sums {
    float m;
    double s, w, s1;
};
template <bool ENTROPY, bool TWO>
__device__ __forceinline__ Sums join_block(Running<ENTROPY, TWO> r, float c, float c1, float* red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m = max_nan(m, red[i]);
    if (!(m <= r.m)) r.raise(m, c, c1);
    const float s = warp_sum(r.s), w = ENTROPY ? warp_sum(r.w) : 0.f, s1 = TWO ? warp_sum(r.s1) : 0.f;
    if (lane == 0) {
        red[WARPS + warp] = s;
        red[2 * WARPS + warp] = w;
        red[3 * WARPS + warp] = s1;
    }
    __syncthreads();
    Sums t{m, 0.0, 0.0, 0.0};
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        t.s += red[WARPS + i];
        if (ENTROPY) t.w += red[2 * WARPS + i];
        if (TWO) t.s1 += red[3 * WARPS + i];
    }
    return t;
}

// ------------------------------------------------------------------ clusters
template <typename V>
__device__ __forceinline__ V ld_peer(const V* p, uint32_t cta) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    V v;
    if constexpr (sizeof(V) == 8) {
        unsigned long long r;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(r) : "r"(a) : "memory");
        v = *reinterpret_cast<V*>(&r);
    } else {
        uint32_t r;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
        v = *reinterpret_cast<V*>(&r);
    }
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------ the k best of a slice
// Values as ordered keys: NaN above everything, zeros of both signs alike.  A candidate is its key above its index
// counted down, so the order of candidates is the order wanted and no two are equal.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return key == 0xffffffffu ? __int_as_float(0x7fffffff) : __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ unsigned long long candidate(uint32_t key, int index) {
    return static_cast<unsigned long long>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int index_of(unsigned long long c) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(c)); }

struct Selection {
    uint32_t group[(SEGMENTS + 1) * THREADS];           // key of the largest value of a thread's share of a segment
    unsigned short chosen[(SEGMENTS + 1) * THREADS];
    unsigned long long cand[MAX_CANDIDATES];
    unsigned long long best[MAX_K];
    uint32_t threshold;
    int groups, count, scan[WARPS];
};

// The first k of the n candidates, in order, into `best`; returns how many there are.  All threads.
__device__ __noinline__ int order_candidates(Selection& sel, int n, int k) {
    const int tid = threadIdx.x;
    if (n <= THREADS) {                                 // everybody counts those ahead of its own
        if (tid < n) {
            const unsigned long long mine = sel.cand[tid];
            int ahead = 0;
            for (int i = 0; i < n; ++i) ahead += sel.cand[i] > mine;
            if (ahead < k) sel.best[ahead] = mine;
        }
    } else {
        int size = 2 * THREADS;
        while (size < n) size *= 2;
        for (int i = n + tid; i < size; i += THREADS) sel.cand[i] = 0;
        __syncthreads();
        for (int width = 2; width <= size; width *= 2)  // bitonic, descending
            for (int gap = width / 2; gap > 0; gap /= 2) {
                for (int i = tid; i < size / 2; i += THREADS) {
                    const int lo = 2 * i - (i & (gap - 1)), hi = lo + gap;
                    const unsigned long long a = sel.cand[lo], b = sel.cand[hi];
                    if ((a < b) == ((lo & width) == 0)) {
                        sel.cand[lo] = b;
                        sel.cand[hi] = a;
                    }
                }
                __syncthreads();
            }
        if (tid < k) sel.best[tid] = sel.cand[tid];
    }
    __syncthreads();
    return min(n, k);
}

// Rows with so many values at or above the first bound that they do not fit (constant rows, above all): the k-th key bit
// by bit with a pass over the slice for each, then those above it, then the first of those equal to it.
template <typename T>
__device__ __noinline__ int select_by_passes(Selection& sel, const Slice<T>& sl, int k) {
    constexpr int N = Elem<T>::N;
    const int tid = threadIdx.x;
    uint32_t bound = 0;
    bool exact = false;
    for (int bit = 31; bit >= 0 && !exact; --bit) {
        const uint32_t trial = bound | 1u << bit;
        int mine = 0;
        for (int j = sl.begin + tid; j < sl.end; j += THREADS) {
            float f[N];
            Elem<T>::unpack(sl.load_any(j), f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int v = sl.index(j, e);
                mine += v >= 0 && v < sl.V && key_of(f[e]) >= trial;
            }
        }
        mine = __reduce_add_sync(0xffffffffu, mine);
        __syncthreads();
        if ((tid & 31) == 0) sel.scan[tid >> 5] = mine;
        __syncthreads();
        int total = 0;
        for (int i = 0; i < WARPS; ++i) total += sel.scan[i];
        if (total >= k) bound = trial;
        exact = total == k;
    }
    if (tid == 0) sel.count = 0;
    __syncthreads();
    for (int j = sl.begin + tid; j < sl.end; j += THREADS) {
        float f[N];
        Elem<T>::unpack(sl.load_any(j), f);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int v = sl.index(j, e);
            const uint32_t key = key_of(f[e]);
            if (v >= 0 && v < sl.V && (exact ? key >= bound : key > bound)) {
                const int at = atomicAdd(&sel.count, 1);        // at most k of them
                if (at < MAX_CANDIDATES) sel.cand[at] = candidate(key, v);
            }
        }
    }
    __syncthreads();
    int have = sel.count;
    for (int j0 = sl.begin; j0 < sl.end && have < k; j0 += THREADS) {     // equal ones, in the order of their indexes
        const int j = j0 + tid;
        float f[N];
        int mine = 0;
        if (j < sl.end) {
            Elem<T>::unpack(sl.load_any(j), f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int v = sl.index(j, e);
                mine += v >= 0 && v < sl.V && key_of(f[e]) == bound;
            }
        }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, upto, o);
            if ((tid & 31) >= o) upto += below;
        }
        if ((tid & 31) == 31) sel.scan[tid >> 5] = upto;
        __syncthreads();
        int at = have + upto - mine, total = 0;
        for (int i = 0; i < WARPS; ++i) {
            if (i < (tid >> 5)) at += sel.scan[i];
            total += sel.scan[i];
        }
        if (mine > 0)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int v = sl.index(j, e);
                if (v >= 0 && v < sl.V && key_of(f[e]) == bound) {
                    if (at < k) sel.cand[at] = candidate(bound, v);
                    ++at;
                }
            }
        have += total;
        __syncthreads();
    }
    return min(have, k);
}

// The k best of a slice, in order, into sel.best; returns how many the slice has.  The stream has left the largest value
// of every group (a thread's vectors of one segment).  At least k values reach the k-th largest of these, and hardly more
// do, so only the groups that reach it are read again: 1.03 k of them where values come in no order.
template <typename T>
__device__ __noinline__ int select_best(Selection& sel, const Slice<T>& sl, int k, int segment_steps) {
    constexpr int N = Elem<T>::N, GROUPS = (SEGMENTS + 1) * THREADS, PER_LANE = GROUPS / 32;
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < 32) {
        uint32_t g[PER_LANE], bound = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) g[i] = sel.group[tid + 32 * i];
        for (int bit = 31; bit >= 32 - Elem<T>::KEY_BITS; --bit) {
            const uint32_t trial = bound | 1u << bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) n += g[i] >= trial;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= k) bound = trial;
            if (n == k) break;
        }
        if (tid == 0) {
            sel.threshold = max(bound, 1u);             // 0: groups without values
            sel.groups = sel.count = 0;
        }
    }
    __syncthreads();
    const uint32_t bound = sel.threshold;
#pragma unroll
    for (int i = 0; i < SEGMENTS + 1; ++i)
        if (sel.group[i * THREADS + tid] >= bound) sel.chosen[atomicAdd(&sel.groups, 1)] = static_cast<unsigned short>(i * THREADS + tid);
    __syncthreads();
    const int per = segment_steps * UNROLL, items = sel.groups * max(per, 1);
    for (int i = tid; i < items; i += THREADS) {
        const int group = sel.chosen[i / max(per, 1)], q = i - i / max(per, 1) * max(per, 1);
        const int segment = group / THREADS, t = group - segment * THREADS;
        int j;
        if (segment == SEGMENTS) {                      // the parts at the row's ends
            if (q > 0) continue;
            j = t == 0 ? 0 : sl.nv - 1;
        } else {
            j = sl.full0 + (segment * per + q) * THREADS + t;
            if (j >= sl.full1) continue;
        }
        float f[N];
        Elem<T>::unpack(sl.load_any(j), f);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t key = key_of(f[e]);
            const int v = sl.index(j, e);
            if (key >= bound && v >= 0 && v < sl.V) {
                const int at = atomicAdd(&sel.count, 1);
                if (at < MAX_CANDIDATES) sel.cand[at] = candidate(key, v);
            }
        }
    }
    __syncthreads();
    int n = sel.count;
    if (n > MAX_CANDIDATES) n = select_by_passes<T>(sel, sl, k);
    __syncthreads();
    return order_candidates(sel, n, k);
}

// ------------------------------------------------------------------ log probabilities, entropies, alternatives
struct ScoreArgs {
    Rows rows;
    const long long* tokens;        // or null
    long long ignore_index;
    double inv_temperature;
    int k, splits;
    float *logprobs, *entropy, *top_logprobs;
    long long* top_ids;
    float* stats;                   // [rows][4]: m, S, entropy, log S; or null
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const __grid_constant__ ScoreArgs p) {
    __shared__ float red[4 * WARPS];
    __shared__ float part_m;
    __shared__ double part_s, part_w, row_log_s;
    __shared__ int part_n;
    __shared__ std::conditional_t<TOP, Selection, int> sel;
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / p.splits;
    const int rank = blockIdx.x - static_cast<int>(r * p.splits);
    const T* row = p.rows.row<T>(r);
    const Slice<T> sl(row, p.rows.V, rank, p.splits);
    const float c = static_cast<float>(p.inv_temperature * 1.4426950408889634);

    Running<true, false> run;
    const int steps = sl.steps(), segment_steps = (steps + SEGMENTS - 1) / SEGMENTS;
    if constexpr (TOP)
        for (int i = 0; i < SEGMENTS + 1; ++i) sel.group[i * THREADS + tid] = 0;
    float largest = -INFINITY;          // of the segment
    bool some = false;
    for (int step = 0, left = segment_steps, segment = 0; step < steps; ++step) {
        uint4 v[UNROLL];
        const int j0 = sl.full0 + step * THREADS * UNROLL + tid;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = j0 + u * THREADS < sl.full1 ? sl.load(j0 + u * THREADS) : Slice<T>::nothing();
        const float m = max_of<T>(v);
        run.template add<T>(v, m, c, 0.f);
        if constexpr (TOP) {
            largest = max_nan(largest, m);
            some |= j0 < sl.full1;
            if (--left == 0 || step == steps - 1) {
                if (some) sel.group[segment * THREADS + tid] = key_of(largest);
                ++segment;
                left = segment_steps;
                largest = -INFINITY;
                some = false;
            }
        }
    }
    if ((tid == 0 && sl.head) || (tid == 1 && sl.tail)) {
        const uint4 v[1] = {sl.load_part(tid == 0 ? 0 : sl.nv - 1)};
        const float m = max_of<T>(v);
        run.template add<T>(v, m, c, 0.f);
        if constexpr (TOP) sel.group[SEGMENTS * THREADS + tid] = key_of(m);
    }
    Sums sum = join_block(run, c, 0.f, red);
    int n = 0;
    if constexpr (TOP) n = select_best<T>(sel, sl, p.k, segment_steps);

    if (p.splits > 1) {
        if (tid == 0) {
            part_m = sum.m;
            part_s = sum.s;
            part_w = sum.w;
            part_n = n;
        }
        cluster_sync();
        if (rank == 0) {
            float m = sum.m;
            for (int q = 0; q < p.splits; ++q) m = max_nan(m, ld_peer(&part_m, q));
            double s = 0, w = 0;
            for (int q = 0; q < p.splits; ++q) {
                const float mq = ld_peer(&part_m, q);
                const double t = mq == m ? 0.0 : fmax(static_cast<double>(mq - m) * c, -1000.0), f = exp2(t);
                const double sq = ld_peer(&part_s, q);
                s += sq * f;
                w += (ld_peer(&part_w, q) + sq * t) * f;
            }
            sum = Sums{m, s, w, 0.0};
            if constexpr (TOP) {
                int base = 0;
                __syncthreads();
                for (int q = 0; q < p.splits; ++q) {
                    const int nq = ld_peer(&part_n, q);
                    for (int i = tid; i < nq; i += THREADS) sel.cand[base + i] = ld_peer(&sel.best[i], q);
                    base += nq;
                }
                __syncthreads();
                n = order_candidates(sel, base, p.k);
            }
        }
    }
    if (rank == 0) {
        if (tid == 0) {
            const double log_s = log(sum.s), entropy = log_s - sum.w / sum.s * LN2;
            if (p.tokens != nullptr) {
                const long long tok = p.tokens[r];
                float lp = 0.f;
                if (tok != p.ignore_index)
                    lp = tok >= 0 && tok < p.rows.V
                             ? static_cast<float>(static_cast<double>(Elem<T>::f(row[tok]) - sum.m) * p.inv_temperature - log_s)
                             : __int_as_float(0x7fffffff);
                p.logprobs[r] = lp;
            }
            p.entropy[r] = static_cast<float>(entropy);
            if (p.stats != nullptr)
                *reinterpret_cast<float4*>(p.stats + 4 * r) = make_float4(
                    sum.m, static_cast<float>(sum.s), static_cast<float>(entropy), static_cast<float>(log_s));
            row_log_s = log_s;
        }
        if constexpr (TOP) {
            __syncthreads();
            if (tid < n) {
                const unsigned long long b = sel.best[tid];
                p.top_ids[r * p.k + tid] = index_of(b);
                p.top_logprobs[r * p.k + tid] = static_cast<float>(
                    static_cast<double>(value_of(static_cast<uint32_t>(b >> 32)) - sum.m) * p.inv_temperature - row_log_s);
            }
        }
    }
    if (p.splits > 1) cluster_sync();   // the leader has read this CTA's part
}

// ------------------------------------------------------------------ gradients
// dx_j = coefficient of the row times the row's exponentials, and other values at single tokens, which overwrite what the
// stream has stored once the CTA has passed a barrier.  A CTA takes one step's vectors of one row: nothing depends on the
// other CTAs, and the loads of many CTAs are in flight together.
template <typename T>
struct GradSlice {
    static constexpr int N = Elem<T>::N;
    Slice<T> in;
    T* out;
    int before, nv, j0;
    bool same;      // rows of both tensors start at the same place of a vector

    // vectors are those of the output; `chunk` of THREADS * UNROLL of them
    __device__ __forceinline__ GradSlice(const T* x, T* out_, int V, int chunk) : in(x, V, 0, 1), out(out_) {
        before = static_cast<int>((reinterpret_cast<uintptr_t>(out_) & 15) / sizeof(T));
        nv = (before + V + N - 1) / N;
        j0 = chunk * THREADS * UNROLL;
        same = before == in.before;
    }
    __device__ __forceinline__ bool has(long long id) const {
        if (id < 0 || id >= in.V) return false;
        const int j = (static_cast<int>(id) + before) / N;
        return j >= j0 && j < j0 + THREADS * UNROLL;
    }
    __device__ __forceinline__ bool whole(int j) const { return j * N >= before && j * N + N - before <= in.V; }
    __device__ __forceinline__ uint4 load(int j) const {
        if (same && whole(j)) return in.load(j);
        uint4 r = Slice<T>::nothing();
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = j * N + i - before;
            if (v >= 0 && v < in.V) e[i] = in.row[v];
        }
        return r;
    }
    __device__ __forceinline__ void store(int j, const float (&f)[N]) const {
        if (whole(j)) {
            *reinterpret_cast<uint4*>(out - before + static_cast<long long>(j) * N) = Elem<T>::pack(f);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = j * N + i - before;
            if (v >= 0 && v < in.V) out[v] = Elem<T>::from(f[i]);
        }
    }
    // out_j = f(x_j)
    template <typename F>
    __device__ __forceinline__ void map(F&& f) const {
        uint4 v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS + threadIdx.x;
            if (j < nv) v[u] = load(j);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS + threadIdx.x;
            if (j < nv) {
                float x[N];
                Elem<T>::unpack(v[u], x);
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = f(x[e]);
                store(j, x);
            }
        }
    }
    __device__ __forceinline__ void zero() const {
        const float z[N] = {};
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS + threadIdx.x;
            if (j < nv) store(j, z);
        }
    }
};

struct ScoreGradArgs {
    Rows rows;
    void* grad;                     // [rows][V], dense
    const long long* tokens;
    long long ignore_index;
    float inv_temperature;
    int k, chunks;
    const float* stats;
    const long long* top_ids;
    const float *d_logprobs, *d_entropy, *d_top;        // any may be null
};

// dx_j = (1 / temperature) (d_tok (1[tok = j] - p_j) - d_ent p_j (log p_j + H) + sum_i d_top_i (1[id_i = j] - p_j))
template <typename T>
__global__ void __launch_bounds__(THREADS) token_logprobs_grad_kernel(const __grid_constant__ ScoreGradArgs p) {
    __shared__ float red[32];
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / p.chunks;
    const int V = p.rows.V;
    T* out = static_cast<T*>(p.grad) + r * V;
    const GradSlice<T> g(p.rows.row<T>(r), out, V, static_cast<int>(blockIdx.x - r * p.chunks));
    const float4 st = *reinterpret_cast<const float4*>(p.stats + 4 * r);
    const float m = st.x, inv_s = 1.f / st.y, c = p.inv_temperature * LOG2E;
    long long tok = -1;
    float d_tok = 0.f;
    if (p.d_logprobs != nullptr) {
        tok = p.tokens[r];
        if (tok == p.ignore_index || tok < 0 || tok >= V) tok = -1;
        else d_tok = p.d_logprobs[r] * p.inv_temperature;
    }
    const float d_ent = p.d_entropy != nullptr ? p.d_entropy[r] * p.inv_temperature : 0.f;
    long long id = -1;
    float d_id = 0.f, d_all = d_tok;
    if (p.d_top != nullptr) {
        if (tid < p.k) {
            id = p.top_ids[r * p.k + tid];
            d_id = p.d_top[r * p.k + tid] * p.inv_temperature;
        }
        d_all += block_sum(d_id, red);
    }
    // p_j (a + b log p_j), log p_j = ln2 t_j - log S
    const float a = -(d_all + d_ent * st.z), b = -d_ent;
    const float a2 = inv_s * (a - b * st.w), b2 = inv_s * b * static_cast<float>(LN2);
    auto value = [&](float x) {
        const float t = max_nan((x - m) * c, T_MIN);
        return exp2_approx(t) * fmaf(b2, t, a2);
    };
    g.map(value);
    bool met = false;
    if (p.d_top != nullptr && id >= 0 && g.has(id)) met = id == tok;
    const bool taken = __syncthreads_or(met);
    if (p.d_top != nullptr && id >= 0 && g.has(id)) out[id] = Elem<T>::from(value(Elem<T>::f(g.in.row[id])) + d_id + (met ? d_tok : 0.f));
    if (tid == 0 && !taken && tok >= 0 && g.has(tok)) out[tok] = Elem<T>::from(value(Elem<T>::f(g.in.row[tok])) + d_tok);
}

// ------------------------------------------------------------------ distillation from a teacher's best tokens
// q: the teacher's listed tokens, and with a tail one bucket for all others, q_r = 1 - sum q.  p: the student, p_r the sum
// over the tokens that are not listed.  KL(q || p) (METHOD 0) or KL(p || q) (METHOD 1) over the buckets.  p_r is summed as
// such and not as 1 - sum p, which would leave nothing of a small rest: the listed tokens are bits of a map in shared memory,
// a byte per vector, and the stream leaves them out.
constexpr double NO_TAIL = 9.5367431640625e-07;     // 2^-20: what 1 - sum q can be by the rounding of fp32 log probabilities

struct DistillArgs {
    Rows rows;
    const long long* ids;           // [rows][k]
    const float* teacher;           // [rows][k] log probabilities (any logits without a tail)
    const long long* labels;        // or null
    long long ignore_index;
    double inv_temperature;
    int k, splits, forward_kl, tail;
    float *kl, *nll;
    int* entries;                   // [rows][k]: the ids that count, -1 elsewhere
    float* stats;                   // [rows][8]
};
// stats: m, 1 / S, factor of p_j at tokens that are not listed, sum q + q_r (METHOD 0) or the loss (METHOD 1), what is taken
// from the teacher's values to make them log probabilities, 1 / S at temperature one, log S, 1 if the row has any loss

struct DistillPart {        // of a CTA, relative to its largest logit m
    float m;
    int n;                  // listed tokens that count
    double rest, top, all1; // sums of exponentials: not listed, listed, all at temperature one
    double q, qx;           // METHOD 0: sum of the teacher's weights u, sum of u (its log - x / temperature)
    double px;              // METHOD 1: sum of listed exponentials times (x / temperature - teacher's log)
};

template <typename T, bool TWO>
__global__ void __launch_bounds__(THREADS, 4) topk_distillation_kernel(const __grid_constant__ DistillArgs p) {
    constexpr int N = Elem<T>::N;
    extern __shared__ __align__(16) uint32_t listed[];      // a byte per vector of this CTA
    __shared__ float red[4 * WARPS];
    __shared__ int id_of[MAX_K];
    __shared__ DistillPart part;
    __shared__ double part_of[WARPS][4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long r = blockIdx.x / p.splits;
    const int rank = blockIdx.x - static_cast<int>(r * p.splits);
    const int V = p.rows.V;
    const T* row = p.rows.row<T>(r);
    const Slice<T> sl(row, V, rank, p.splits);
    const float c = static_cast<float>(p.inv_temperature * 1.4426950408889634);

    // the list: entries that count are in the vocabulary, have a finite or NaN value, and come first of their token
    int id = -1;
    float lq = -INFINITY;
    if (tid < p.k) {
        const long long i = p.ids[r * p.k + tid];
        lq = p.teacher[r * p.k + tid];
        if (i >= 0 && i < V && lq != -INFINITY) id = static_cast<int>(i);
        id_of[tid] = id;
    }
    const long long label = p.labels != nullptr ? p.labels[r] : p.ignore_index;
    const bool labelled = label != p.ignore_index;
    const bool any = __syncthreads_or(id >= 0);
    if (!any && !labelled) {            // nothing is asked of this row: it is not read
        if (rank == 0) {
            if (tid < p.k) p.entries[r * p.k + tid] = -1;
            if (tid == 0) {
                p.kl[r] = 0.f;
                if (p.nll != nullptr) p.nll[r] = 0.f;
            }
            if (tid < 8) p.stats[8 * r + tid] = 0.f;
        }
        return;                         // (all CTAs of the cluster alike)
    }
    const int words = (sl.end - sl.begin + 3) / 4;
    for (int i = tid; i < words; i += THREADS) listed[i] = 0;
    __syncthreads();
    const bool mine = id >= 0 && sl.has(id);
    bool again = false;
    if (mine) {
        const int j = (id + sl.before) / N - sl.begin, bit = (j & 3) * 8 + (id + sl.before) % N;
        again = atomicOr(&listed[j >> 2], 1u << bit) >> bit & 1u;
    }
    bool counts = mine;
    if (__syncthreads_or(again) && mine)
        for (int i = 0; i < tid; ++i) counts &= id_of[i] != id;
    if (tid < p.k && (mine || (rank == 0 && id < 0))) p.entries[r * p.k + tid] = counts ? id : -1;

    Running<false, TWO> run;
    const uint8_t* flag = reinterpret_cast<const uint8_t*>(listed);
    const int steps = sl.steps();
    auto hide = [&](uint4& v, int j) {
        const uint32_t b = flag[j - sl.begin];
        if (b != 0) {
            T* e = reinterpret_cast<T*>(&v);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (b >> i & 1u) e[i] = Elem<T>::from(-INFINITY);
        }
    };
    for (int step = 0; step < steps; ++step) {
        uint4 v[UNROLL];
        const int j0 = sl.full0 + step * THREADS * UNROLL + tid;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = j0 + u * THREADS < sl.full1 ? sl.load(j0 + u * THREADS) : Slice<T>::nothing();
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (j0 + u * THREADS < sl.full1) hide(v[u], j0 + u * THREADS);
        run.template add<T>(v, max_of<T>(v), c, LOG2E);
    }
    if ((tid == 0 && sl.head) || (tid == 1 && sl.tail)) {
        const int j = tid == 0 ? 0 : sl.nv - 1;
        uint4 v[1] = {sl.load_part(j)};
        hide(v[0], j);
        run.template add<T>(v, max_of<T>(v), c, LOG2E);
    }
    Sums sum = join_block(run, c, LOG2E, red);

    // the listed tokens, in 64 bits.  Weights without a tail are relative to the largest value of the list.
    const float x = counts ? Elem<T>::f(row[id]) : -INFINITY;
    float m = max_nan(x, -INFINITY), ref = id >= 0 ? lq : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        ref = max_nan(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    }
    __syncthreads();
    if (lane == 0) {
        red[warp] = m;
        red[WARPS + warp] = ref;
    }
    __syncthreads();
    for (int i = 0; i < MAX_K / 32; ++i) {
        m = max_nan(m, red[i]);
        ref = max_nan(ref, red[WARPS + i]);
    }
    m = max_nan(m, sum.m);
    if (p.tail || ref == -INFINITY) ref = 0.f;
    double e[4] = {0, 0, 0, 0};         // listed exponentials, at temperature one, weights, products
    if (counts) {
        const double d = static_cast<double>(x) - m, y = static_cast<double>(x) * p.inv_temperature;
        e[0] = x == -INFINITY ? 0.0 : exp(d * p.inv_temperature);
        e[1] = TWO ? (x == -INFINITY ? 0.0 : exp(d)) : 0.0;
        e[2] = exp(static_cast<double>(lq) - ref);
        if (p.forward_kl) e[3] = e[0] == 0.0 ? 0.0 : e[0] * (y - lq);
        else e[3] = e[2] == 0.0 ? 0.0 : e[2] * (static_cast<double>(lq) - ref - y);
    }
    if (warp < MAX_K / 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) e[q] += __shfl_xor_sync(0xffffffffu, e[q], o);
        if (lane == 0)
            for (int q = 0; q < 4; ++q) part_of[warp][q] = e[q];
    }
    const int n = __syncthreads_count(counts);
    if (tid == 0) {
        for (int q = 0; q < 4; ++q) {
            e[q] = 0;
            for (int i = 0; i < MAX_K / 32; ++i) e[q] += part_of[i][q];
        }
        const double d = sum.m == m ? 0.0 : fmax(static_cast<double>(sum.m) - m, -1e30);
        const double f = exp(d * p.inv_temperature);
        part = DistillPart{m, n, sum.s * f, e[0], TWO ? sum.s1 * exp(d) + e[1] : 0.0, e[2], p.forward_kl ? 0.0 : e[3],
                           p.forward_kl ? e[3] : 0.0};
    }
    if (p.splits > 1) cluster_sync();
    if (rank == 0 && tid == 0) {
        DistillPart all = part;
        if (p.splits > 1) {
            for (int q = 1; q < p.splits; ++q) all.m = max_nan(all.m, ld_peer(&part.m, q));
            all.n = 0;
            all.rest = all.top = all.all1 = all.q = all.qx = all.px = 0;
            for (int q = 0; q < p.splits; ++q) {
                const float mq = ld_peer(&part.m, q);
                const double d = mq == all.m ? 0.0 : fmax(static_cast<double>(mq) - all.m, -1e30);
                const double f = exp(d * p.inv_temperature);
                all.n += ld_peer(&part.n, q);
                all.rest += ld_peer(&part.rest, q) * f;
                all.top += ld_peer(&part.top, q) * f;
                all.px += ld_peer(&part.px, q) * f;
                if (TWO) all.all1 += ld_peer(&part.all1, q) * exp(d);
                all.q += ld_peer(&part.q, q);
                all.qx += ld_peer(&part.qx, q);
            }
        }
        const double S = all.rest + all.top, log_s = log(S), lse = all.m * p.inv_temperature + log_s;
        const double S1 = TWO ? all.all1 : S;
        double kl = 0, factor = 0, fourth = 0, norm = 0;
        if (all.n > 0) {
            const double p_r = all.rest / S, log_p_r = log(p_r);
            double q_r = 0;
            if (p.tail) {
                q_r = 1 - all.q;
                if (q_r < NO_TAIL) q_r = 0;
            }
            if (!p.forward_kl) {
                if (p.tail) {
                    kl = all.qx + all.q * lse;
                    if (q_r > 0) kl += q_r * (log(q_r) - log_p_r);
                    fourth = all.q + q_r;
                } else {
                    norm = ref + log(all.q);
                    kl = all.qx / all.q - log(all.q) + lse;
                    fourth = 1;
                }
                factor = fourth - (p_r > 0 ? q_r / p_r : 0.0);
            } else {
                const double ratio = p_r > 0 ? log_p_r - log(fmax(q_r, NO_TAIL)) : 0.0;
                kl = (all.px - all.top * lse) / S + p_r * ratio;
                fourth = kl;
                factor = ratio - kl;
            }
        }
        p.kl[r] = static_cast<float>(kl);
        if (p.nll != nullptr)
            p.nll[r] = !labelled ? 0.f
                       : label >= 0 && label < V
                           ? static_cast<float>(log(S1) - (static_cast<double>(Elem<T>::f(row[label])) - all.m))
                           : __int_as_float(0x7fffffff);
        float4* st = reinterpret_cast<float4*>(p.stats + 8 * r);
        st[0] = make_float4(all.m, static_cast<float>(1 / S), static_cast<float>(factor), static_cast<float>(fourth));
        st[1] = make_float4(static_cast<float>(norm), static_cast<float>(1 / S1), static_cast<float>(log_s), 1.f);
    }
    if (p.splits > 1) cluster_sync();
}

struct DistillGradArgs {
    Rows rows;
    void* grad;
    const int* entries;
    const float* teacher;
    const long long* labels;
    long long ignore_index;
    float inv_temperature;
    int k, chunks, forward_kl;
    const float* stats;
    const float *d_kl, *d_nll;      // either may be null
};

// Tokens that are not listed: p_j times the row's factor.  Listed ones: p_i (sum q + q_r) - q_i (METHOD 0),
// p_i (log p_i - log q_i - KL) (METHOD 1).  Both over the temperature, and the cross entropy's p_j - 1[label = j] on top.
template <typename T, bool TWO>
__global__ void __launch_bounds__(THREADS) topk_distillation_grad_kernel(const __grid_constant__ DistillGradArgs p) {
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / p.chunks;
    const int V = p.rows.V;
    T* out = static_cast<T*>(p.grad) + r * V;
    const GradSlice<T> g(p.rows.row<T>(r), out, V, static_cast<int>(blockIdx.x - r * p.chunks));
    const float4 s0 = reinterpret_cast<const float4*>(p.stats + 8 * r)[0], s1 = reinterpret_cast<const float4*>(p.stats + 8 * r)[1];
    if (s1.w == 0.f) {              // no loss: not read, gradient zero
        g.zero();
        return;
    }
    const float m = s0.x, inv_s = s0.y, c = p.inv_temperature * LOG2E;
    const float d_kl = p.d_kl != nullptr ? p.d_kl[r] * p.inv_temperature : 0.f;
    long long label = -1;
    float d_nll = 0.f;
    if (p.d_nll != nullptr) {
        label = p.labels[r];
        if (label == p.ignore_index || label < 0 || label >= V) label = -1;
        else d_nll = p.d_nll[r];
    }
    const float a = d_kl * inv_s * s0.z + (TWO ? 0.f : d_nll * inv_s), a1 = d_nll * s1.y;
    auto t_of = [&](float x) { return max_nan((x - m) * c, T_MIN); };
    auto e1_of = [&](float x) { return exp2_approx(max_nan((x - m) * LOG2E, T_MIN)); };
    auto value = [&](float x) {
        const float v = exp2_approx(t_of(x)) * a;
        return TWO ? fmaf(e1_of(x), a1, v) : v;
    };
    g.map(value);
    int id = -1;
    if (tid < p.k) id = p.entries[r * p.k + tid];
    const bool here = id >= 0 && g.has(id), met = here && id == label;
    const bool taken = __syncthreads_or(met);
    if (here) {
        const float x = Elem<T>::f(g.in.row[id]), t = t_of(x), e = exp2_approx(t) * inv_s;
        const float lq = p.teacher[r * p.k + tid] - s1.x;
        float v;
        if (p.forward_kl) v = e == 0.f ? 0.f : e * (t * static_cast<float>(LN2) - s1.z - lq - s0.w);
        else v = e * s0.w - __expf(lq);
        v = v * d_kl + d_nll * (TWO ? e1_of(x) * s1.y : e) - (met ? d_nll : 0.f);
        out[id] = Elem<T>::from(v);
    }
    if (tid == 0 && !taken && label >= 0 && g.has(label)) out[label] = Elem<T>::from(value(Elem<T>::f(g.in.row[label])) - d_nll);
}

// ------------------------------------------------------------------ launches
// CTAs per row: one when there are rows for every SM, else as many as it takes to give each SM about two, while a CTA
// keeps a step of work.
inline int splits_for(long long rows, int V, int elem) {
    const int step = THREADS * 16 / elem;
    int n = 1;
    while (n < MAX_SPLITS && rows * n < 296 && V > step * n) n *= 2;
    return n;
}

template <typename Kern, typename Args>
inline cudaError_t launch(Kern kern, const Args& a, long long ctas, int splits, int smem, void* stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

inline int elem_size(int dtype) { return dtype == LME_F32 ? 4 : 2; }
inline int chunks_for(int V, int elem) {     // of a gradient row, whose first vector may be a part
    const int n = 16 / elem;
    return (V + 2 * n - 2 + n * THREADS * UNROLL - 1) / (n * THREADS * UNROLL);
}
constexpr long long MAX_GRID = 0x7fffffff;
constexpr int MAX_V = 1 << 30;

}  // namespace vr
}  // namespace lme

extern "C" int lme_token_logprobs_fwd(const void* x, int dtype, long long rows, long long inner, long long ld_inner,
                                      long long ld_outer, int V, const long long* tokens, long long ignore_index,
                                      double temperature, int k, float* logprobs, float* entropy, float* top_logprobs,
                                      long long* top_ids, float* stats, void* stream) {
    using namespace lme::vr;
    if (dtype < LME_BF16 || dtype > LME_F32 || rows < 0 || inner < 1 || V < 1 || k < 0 || k > MAX_K || k > V || !(temperature > 0))
        return LME_ERR_SHAPE;
    if (rows == 0) return LME_OK;
    const int splits = splits_for(rows, V, elem_size(dtype));
    if (V > MAX_V || rows * splits > MAX_GRID) return LME_ERR_TOO_LARGE;
    const ScoreArgs a{{x, inner, ld_inner, ld_outer, V}, tokens, ignore_index, 1.0 / temperature, k, splits, logprobs, entropy,
                      top_logprobs, top_ids, stats};
    const long long ctas = rows * splits;
    cudaError_t e;
    if (dtype == LME_BF16)
        e = k > 0 ? launch(token_logprobs_kernel<__nv_bfloat16, true>, a, ctas, splits, 0, stream)
                  : launch(token_logprobs_kernel<__nv_bfloat16, false>, a, ctas, splits, 0, stream);
    else if (dtype == LME_F16)
        e = k > 0 ? launch(token_logprobs_kernel<__half, true>, a, ctas, splits, 0, stream)
                  : launch(token_logprobs_kernel<__half, false>, a, ctas, splits, 0, stream);
    else
        e = k > 0 ? launch(token_logprobs_kernel<float, true>, a, ctas, splits, 0, stream)
                  : launch(token_logprobs_kernel<float, false>, a, ctas, splits, 0, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}

extern "C" int lme_token_logprobs_bwd(const void* x, int dtype, long long rows, long long inner, long long ld_inner,
                                      long long ld_outer, int V, const long long* tokens, long long ignore_index,
                                      double temperature, int k, const float* stats, const long long* top_ids,
                                      const float* d_logprobs, const float* d_entropy, const float* d_top, void* grad,
                                      void* stream) {
    using namespace lme::vr;
    if (dtype < LME_BF16 || dtype > LME_F32 || rows < 0 || inner < 1 || V < 1 || k < 0 || k > MAX_K || !(temperature > 0) ||
        (d_logprobs != nullptr && tokens == nullptr))
        return LME_ERR_SHAPE;
    if (rows == 0) return LME_OK;
    const int chunks = chunks_for(V, elem_size(dtype));
    if (V > MAX_V || rows * chunks > MAX_GRID) return LME_ERR_TOO_LARGE;
    const ScoreGradArgs a{{x, inner, ld_inner, ld_outer, V}, grad, tokens, ignore_index, static_cast<float>(1.0 / temperature), k,
                          chunks, stats, top_ids, d_logprobs, d_entropy, d_top};
    const long long ctas = rows * chunks;
    const cudaError_t e = dtype == LME_BF16  ? launch(token_logprobs_grad_kernel<__nv_bfloat16>, a, ctas, 1, 0, stream)
                          : dtype == LME_F16 ? launch(token_logprobs_grad_kernel<__half>, a, ctas, 1, 0, stream)
                                             : launch(token_logprobs_grad_kernel<float>, a, ctas, 1, 0, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}

namespace lme {
namespace vr {
template <typename T>
inline cudaError_t launch_distill(const DistillArgs& a, bool two, long long ctas, int splits, int smem, void* stream) {
    if (smem > 48 * 1024) {
        const bool ok = two ? opt_in<topk_distillation_kernel<T, true>>(cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_MAP)
                            : opt_in<topk_distillation_kernel<T, false>>(cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_MAP);
        if (!ok) return cudaErrorInvalidValue;
    }
    return two ? launch(topk_distillation_kernel<T, true>, a, ctas, splits, smem, stream)
               : launch(topk_distillation_kernel<T, false>, a, ctas, splits, smem, stream);
}
template <typename T>
inline cudaError_t launch_distill_grad(const DistillGradArgs& a, bool two, long long ctas, void* stream) {
    return two ? launch(topk_distillation_grad_kernel<T, true>, a, ctas, 1, 0, stream)
               : launch(topk_distillation_grad_kernel<T, false>, a, ctas, 1, 0, stream);
}
}  // namespace vr
}  // namespace lme

extern "C" int lme_topk_distillation_fwd(const void* x, int dtype, long long rows, long long inner, long long ld_inner,
                                         long long ld_outer, int V, const long long* top_ids, const float* top_logprobs, int k,
                                         const long long* labels, long long ignore_index, double temperature, int forward_kl,
                                         int tail, float* kl, float* nll, int* entries, float* stats, void* stream) {
    using namespace lme::vr;
    if (dtype < LME_BF16 || dtype > LME_F32 || rows < 0 || inner < 1 || V < 1 || k < 1 || k > MAX_K || !(temperature > 0) ||
        (forward_kl && !tail) || (labels != nullptr) != (nll != nullptr))
        return LME_ERR_SHAPE;
    if (rows == 0) return LME_OK;
    const int n = 16 / elem_size(dtype);
    int splits = splits_for(rows, V, elem_size(dtype));
    auto map_bytes = [&](int s) { return (((V + 2 * n - 2) / n + s - 1) / s + 3 + 16) / 16 * 16; };
    if (V > MAX_V) return LME_ERR_TOO_LARGE;
    while (splits < MAX_SPLITS && map_bytes(splits) > MAX_MAP) splits *= 2;
    if (map_bytes(splits) > MAX_MAP || rows * splits > MAX_GRID) return LME_ERR_TOO_LARGE;
    const DistillArgs a{{x, inner, ld_inner, ld_outer, V}, top_ids, top_logprobs, labels, ignore_index, 1.0 / temperature, k,
                        splits, forward_kl, tail, kl, nll, entries, stats};
    const bool two = labels != nullptr && temperature != 1.0;
    const long long ctas = rows * splits;
    const int smem = map_bytes(splits);
    const cudaError_t e = dtype == LME_BF16  ? launch_distill<__nv_bfloat16>(a, two, ctas, splits, smem, stream)
                          : dtype == LME_F16 ? launch_distill<__half>(a, two, ctas, splits, smem, stream)
                                             : launch_distill<float>(a, two, ctas, splits, smem, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}

extern "C" int lme_topk_distillation_bwd(const void* x, int dtype, long long rows, long long inner, long long ld_inner,
                                         long long ld_outer, int V, const int* entries, const float* top_logprobs, int k,
                                         const long long* labels, long long ignore_index, double temperature, int forward_kl,
                                         const float* stats, const float* d_kl, const float* d_nll, void* grad, void* stream) {
    using namespace lme::vr;
    if (dtype < LME_BF16 || dtype > LME_F32 || rows < 0 || inner < 1 || V < 1 || k < 1 || k > MAX_K || !(temperature > 0) ||
        (d_nll != nullptr && labels == nullptr))
        return LME_ERR_SHAPE;
    if (rows == 0) return LME_OK;
    const int chunks = chunks_for(V, elem_size(dtype));
    if (V > MAX_V || rows * chunks > MAX_GRID) return LME_ERR_TOO_LARGE;
    const DistillGradArgs a{{x, inner, ld_inner, ld_outer, V}, grad, entries, top_logprobs, labels, ignore_index,
                            static_cast<float>(1.0 / temperature), k, chunks, forward_kl, stats, d_kl, d_nll};
    const bool two = d_nll != nullptr && temperature != 1.0;
    const long long ctas = rows * chunks;
    const cudaError_t e = dtype == LME_BF16  ? launch_distill_grad<__nv_bfloat16>(a, two, ctas, stream)
                          : dtype == LME_F16 ? launch_distill_grad<__half>(a, two, ctas, stream)
                                             : launch_distill_grad<float>(a, two, ctas, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}
