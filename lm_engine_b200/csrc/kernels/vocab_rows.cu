// Rows of logits over a vocabulary: log probabilities of given tokens with entropies and the best alternatives, and the
// distillation loss against a teacher's best tokens, each with the gradient of the logits.
//
// With y = x / temperature, m the row's largest logit and t_j = (x_j - m) / temperature, everything that a row needs is
//   S = sum exp(t_j),   W = sum exp(t_j) t_j,   log p_j = t_j - log S,   entropy = log S - W / S
// and a handful of single logits.  The exponent is a difference taken in one rounding or before the product, so no large
// numbers meet in it, whatever the temperature; sums run in fp32 per thread and over the lanes of a warp, warps and CTAs are
// joined in 64 bits, where the few values per row are finished too.
// Fewer bits on purpose: an exponential is the hardware's 2^t (2^-22 off) of an exponent in fp32, since the exponential unit is
// what binds a stream next (75 % busy), and what goes from a forward to its backward kernel is fp32.  Rows that a few tokens
// dominate show it in their entropies, because those tokens' terms are not exactly one (the base follows the largest logit at a
// distance, see Running).  Entropies relative to 64 bits, root mean square and worst, next to elementary fp32 operations that take
// the largest logit away first: 300 single rows of 128256 bf16 logits at temperature 0.7 8e-7 and 5e-6 (3e-7, 1.4e-6), 24 rows of
// 50257 fp32 logits 9e-8 and 7e-7 (1.1e-7, 3e-7), 333 rows of 32000 bf16 logits 2.2e-7 and 1.6e-6 (1.1e-7, 5e-7); log probabilities
// absolutely 3.3e-7, 2.1e-7 and 2.4e-7 (5.8e-7, 2.7e-7, 2.3e-7).  Joining a warp's lanes in 64 bits too changes none of these.
//
// Bound by HBM (one read of the logits forward, a read and a write backward) and, sustained, by the power that the
// instructions per logit take: a CTA of 128 threads streams a row through rings of bulk copies, one per warp; rows are split
// over a cluster of up to 8 CTAs when there are few of them, and joined through distributed shared memory: one launch, no
// workspace, a fixed order of sums.
// Measured on a B200 (1000 W, sustained; up to 12 % more or less on others): scores of 4094 x 128256 bf16 logits 184 us
// = 5.7 TB/s, with the best 64 of 4096 rows 238 us = 4.4 TB/s; gradient at 4096 x 128256 328 us = 6.4 TB/s;
// distillation at 8192 x 128256 with the best 64, forward 344 us = 6.1 TB/s, backward 644 us = 6.5 TB/s.
// Included by lme_cuda.cu after decode_attention.cu.
#include <cuda_fp16.h>

namespace lme {
namespace vr {

constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int UNROLL = 4;               // vectors of 16 bytes per thread and step
constexpr int WARP_STEP = 32 * UNROLL;  // vectors of a warp and step
constexpr int RING_STAGES = 2;
constexpr int RING_BYTES = WARPS * RING_STAGES * WARP_STEP * 16;
constexpr int MAX_SPLITS = 8;           // CTAs of a cluster
constexpr int MAX_K = LME_VOCAB_MAX_K;  // best tokens, or tokens of a teacher, per row
constexpr int SEGMENTS = 16;            // of a CTA's steps: what the selection reads again goes by their maxima
constexpr int MAX_CANDIDATES = 1024;
constexpr int MAX_MAP = 96 * 1024;      // bytes of the map of listed tokens, a byte for each vector of a CTA
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
// two fp32 values per instruction: the stream is bound by its instructions about as much as by HBM
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(unsigned long long p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int N = 8;         // per vector
    static constexpr uint32_t NEG_INF = 0xff80ff80u;
    static constexpr uint32_t LOW2 = 0xf14af14au;       // two of LOW
    static constexpr float LOW = -1.00025555e30f;
    static __device__ __forceinline__ float f(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
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
    static constexpr uint32_t NEG_INF = 0xfc00fc00u;
    static constexpr uint32_t LOW2 = 0xfbfffbffu;
    static constexpr float LOW = -65504.f;
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

// element i of a vector, in registers or shared memory (by bytes: the two types may not alias)
template <typename T>
__device__ __forceinline__ void put(uint4& v, int i, T x) {
    memcpy(reinterpret_cast<unsigned char*>(&v) + i * sizeof(T), &x, sizeof(T));
}
template <typename T>
__device__ __forceinline__ T get(const uint4& v, int i) {
    T x;
    memcpy(&x, reinterpret_cast<const unsigned char*>(&v) + i * sizeof(T), sizeof(T));
    return x;
}

// ------------------------------------------------------------------ rows and their slices
// Row r starts at x + (r / inner) * ld_outer + (r % inner) * ld_inner: sequences whose last positions are left out are
// read in place.
struct Rows {
    const void* x;
    long long inner, ld_inner, ld_outer;
    int V;
    template <typename T>
    __device__ __forceinline__ const T* row(long long r) const {
        if (r < inner) return static_cast<const T*>(x) + r * ld_inner;
        const unsigned o = static_cast<unsigned>(r) / static_cast<unsigned>(inner);     // (at most 2^31 rows)
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
        const int per = splits == 1 ? nv : (nv + splits - 1) / splits;
        begin = min(nv, rank * per);
        end = min(nv, begin + per);
        const bool ragged = (before + V) % N != 0;
        head = begin == 0 && end > 0 && (before > 0 || (nv == 1 && ragged));
        tail = end == nv && end > begin && nv > 1 && ragged;
        full0 = begin + (head ? 1 : 0);
        full1 = end - (tail ? 1 : 0);
    }
    __device__ __forceinline__ int index(int j, int e) const { return j * N + e - before; }
    __device__ __forceinline__ int size() const {           // values of this CTA
        return max(0, min(V, end * N - before) - max(0, begin * N - before));
    }
    __device__ __forceinline__ bool has(int id) const {     // whether token `id` is in this CTA's vectors
        const int j = (id + before) / N;
        return id >= 0 && id < V && j >= begin && j < end;
    }
    __device__ __forceinline__ const T* at(int j) const { return row - before + static_cast<long long>(j) * N; }
    __device__ __forceinline__ uint4 load(int j) const {    // a whole vector
        const T* p = at(j);
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
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = index(j, i);
            if (v >= 0 && v < V) put(r, i, row[v]);
        }
        return r;
    }
    __device__ __forceinline__ bool whole(int j) const { return j >= full0 && j < full1; }
    __device__ __forceinline__ uint4 load_any(int j) const { return whole(j) ? load(j) : load_part(j); }
    __device__ __forceinline__ int steps() const { return (full1 - full0 + THREADS * UNROLL - 1) / (THREADS * UNROLL); }
};

// A warp's whole vectors arrive in a ring of its own, two steps of 2 KB that one lane requests ahead: the loads in
// flight take no registers, and no warp waits for another.
template <typename T>
struct Ring {
    static constexpr uint32_t BYTES = WARP_STEP * 16;
    // Shared addresses of this warp's stages and barriers.  These have memory of their own, which nothing else is ever put into:
    // a barrier's words may serve another purpose only after mbarrier.inval (without it they came back over ordinary stores).
    uint32_t buf, full;
    const T* source;        // of the next request
    int steps;              // those in which this warp has vectors
    int last;               // vectors of the last one
    int ahead;              // requests so far
    bool ok;

    __device__ __forceinline__ Ring(const Slice<T>& sl, uint8_t* smem, uint64_t* barriers) : ahead(0), ok(true) {
        const int warp = threadIdx.x >> 5;
        buf = smem_u32(smem) + warp * RING_STAGES * BYTES;
        uint64_t* bars = barriers + warp * RING_STAGES;
        full = smem_u32(bars);
        const int j = sl.full0 + warp * WARP_STEP;
        steps = j < sl.full1 ? (sl.full1 - j - 1) / (THREADS * UNROLL) + 1 : 0;
        last = min(WARP_STEP, sl.full1 - j - (steps - 1) * (THREADS * UNROLL));
        source = sl.at(j);
        if ((threadIdx.x & 31) == 0) {
            for (int i = 0; i < RING_STAGES; ++i) mbar_init(bars + i, 1);
            fence_barrier_init();
            for (int i = 0; i < RING_STAGES; ++i) request(i);
        }
        __syncwarp();
    }
    // one lane: the next step into a slot, if there is one
    __device__ __forceinline__ void request(int slot) {
        if (ahead >= steps) return;
        const uint32_t bytes = ++ahead == steps ? last * 16 : BYTES;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * slot), "r"(bytes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(buf + slot * BYTES),
                     "l"(source), "r"(bytes), "r"(full + 8 * slot)
                     : "memory");
        source += THREADS * UNROLL * Elem<T>::N;
    }
    static __device__ __forceinline__ uint4 ld(uint32_t address) {
        uint4 r;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(address) : "memory");
        return r;
    }
    // f(step, vectors, whether all of them are there) for every step; nothing behind the last whole vector.  first(step,
    // address): before a lane reads its vectors, 512 bytes apart from `address` on.  After a wait that ran out (status word set)
    // the loop goes on with what the stages hold and requests nothing more; `ok` says that all has arrived.
    template <typename F0, typename F>
    __device__ __forceinline__ void stream(F0&& first, F&& f) {
        const int lane = threadIdx.x & 31;
        for (int step = 0, slot = 0, phase = 0; step < steps; ++step) {
            if (ok) ok = wait(full + 8 * slot, phase);
            const uint32_t b = buf + slot * BYTES + lane * 16;
            first(step, b);
            uint4 v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) v[u] = ld(b + 512 * u);
            const bool whole = step < steps - 1 || last == WARP_STEP;
            if (!whole)
#pragma unroll
                for (int u = 0; u < UNROLL; ++u)
                    if (lane + 32 * u >= last) v[u] = Slice<T>::nothing();      // (and not what the slot held)
            f(step, v, whole);
            // A bulk copy writes through the async proxy, which no barrier of the warp orders behind ordinary reads: every lane's
            // fence does.  (Without one a stage that was requested right behind its reads was overwritten under them.)
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && ok) request(slot);
            if (++slot == RING_STAGES) {
                slot = 0;
                phase ^= 1;
            }
        }
        if (!ok) drain();
    }
    // Waits for what has been requested and not used: no copy may outlast its CTA.  Only the lane that requests knows how
    // much that is; a slot's last request completes its phase number (ahead - 1 - slot) / RING_STAGES.
    __device__ __forceinline__ void drain() {
        if ((threadIdx.x & 31) == 0)
            for (int i = 0; i < min(RING_STAGES, ahead); ++i) wait(full + 8 * i, (ahead - 1 - i) / RING_STAGES & 1);
    }

private:
    static __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
        uint32_t there;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t"
            "}\n"
            : "=r"(there)
            : "r"(bar), "r"(parity)
            : "memory");
        if (there) return true;
        return mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity, 620);
    }
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
// m: a base that no logit so far is above by more than SLACK / c, s: sum of 2^t, w: sum of 2^t t with t = (x - m) c.  The base
// follows the largest logit only past the slack: a thread meets a new largest in most of its steps at first, and its warp with
// it, but few that are so much larger.  A NaN reaches all three.
//
// That is nine instructions per logit, and sustained the power limit makes each of them cost time.  So after a first step
// that sets the base, steps are tried in three and a half: t = x c - n in one rounding, n an integer next to m c (units of 2^n
// until leave()), no largest logit and no guard for minus infinity, and the sums are looked at afterwards; where they have run
// over or are NaN the step is done again in the careful way, and the rest of the row too.
constexpr float SLACK = 8.f;
constexpr float TRY_BELOW = 1.2676506e30f;              // 2^100
// AtOne: how the sum at temperature one is found beside the other: not at all, by exponentials of its own (as many again, and the
// exponential unit is what bounds the stream then), or at temperature two by squares.  Distillation of 4096 x 128256
// bf16 logits at temperature two, forward: 275 us with exponentials of their own, 200 with squares.
enum AtOne { NONE, OWN, SQUARE };
template <bool ENTROPY, AtOne ONE>
struct Running {
    float m = -INFINITY, limit = -INFINITY;
    // s and w, and what their additions have lost.  Vectors, then steps are added up by themselves: next to a token that the model
    // is sure of, single small terms would be lost in its thread's sums, all of them downwards (entropies of 128256 logits at
    // temperature 0.8: off by 1.1e-5 on average, so by 2e-7; 2 to 3 % of the time).
    float s = 0.f, w = 0.f, s_lost = 0.f, w_lost = 0.f;
    float s1 = 0.f;                 // s at temperature one (c1)
    bool far = false;               // 16-bit types: LOW is so far below the base that it counts nothing
    bool trying = false, tried = false;
    float n = 0.f, n1 = 0.f;        // while trying

    // to another unit, 2^by times smaller
    __device__ __forceinline__ void change(float by, float f) {
        if (ENTROPY) {
            w = (w + s * by) * f;
            w_lost = (w_lost + s_lost * by) * f;
        }
        s *= f;
        s_lost *= f;
    }
    __device__ __forceinline__ void raise(float to, float c, float c1) {
        const float d = m - to;
        const float t = max_nan(d * c, T_MIN);          // (-inf) - (-inf) cannot be: `to` is above m
        change(t, exp2_approx(t));
        if (ONE) s1 *= exp2_approx(max_nan(d * c1, T_MIN));
        m = to;
        limit = to + __fdividef(SLACK, ONE ? fmaxf(c, c1) : c);
    }
    // from units of 2^(m c) to those of 2^n
    __device__ __forceinline__ void enter(float c, float c1) {
        if (m == -INFINITY) return;                     // (no base yet)
        tried = true;
        if (!(fabsf(m) * (ONE == OWN ? fmaxf(c, c1) : c) < 1e6f)) return;
        n = rintf(m * c);
        const float by = fmaf(m, c, -n), f = exp2_approx(by);
        change(by, f);
        if (ONE == SQUARE) s1 *= f * f;
        if (ONE == OWN) {
            n1 = rintf(m * c1);
            s1 *= exp2_approx(fmaf(m, c1, -n1));
        }
        trying = true;
    }
    __device__ __forceinline__ void leave(float c, float c1) {
        if (!trying) return;
        const float by = -fmaf(m, c, -n), f = exp2_approx(by);
        change(by, f);
        if (ONE == SQUARE) s1 *= f * f;
        if (ONE == OWN) s1 *= exp2_approx(-fmaf(m, c1, -n1));
        trying = false;
    }
    // At the end, for entropies: the base moves to where the thread's sum is about one, before w is rounded to what is left of
    // it.  In 64 bits: the two terms of the new w are much larger than it.
    __device__ __forceinline__ void settle(float c) {
        if (!(s > 0.f && s < INFINITY)) {
            leave(c, 0.f);
            return;
        }
        float l;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(l) : "f"(s));
        l = rintf(l);
        const float to = trying ? __fdividef(n + l, c) : m + __fdividef(l, c);
        const float by = trying ? fmaf(to, c, -(n + l)) : fmaf(to - m, c, -l);      // beside the power of two
        if (!(fabsf(by) < 1.f)) {                       // (bases too large for such steps)
            leave(c, 0.f);
            return;
        }
        const double s_ = static_cast<double>(s) - s_lost, w_ = static_cast<double>(w) - w_lost;
        const double f = exp2_approx(-by) * __int_as_float((127 - static_cast<int>(fmaxf(fminf(l, 120.f), -120.f))) << 23);
        w = static_cast<float>((w_ - s_ * (static_cast<double>(l) + by)) * f);
        s = static_cast<float>(s_ * f);
        s_lost = w_lost = 0.f;
        m = to;
        trying = false;
    }
    // whole: no vector of the step is filled up; largest(): of the step
    template <typename T, int U, typename F>
    __device__ __forceinline__ void add(const uint4 (&r)[U], bool whole, F&& largest, float c, float c1) {
        if (trying) {
            if (whole && sum<T, U, true, false, false>(r, c, c1)) return;
            leave(c, c1);
        }
        const float x = largest();
        if (!(x <= limit)) {
            raise(x, c, c1);
            if constexpr (Elem<T>::N == 8) far = m - Elem<T>::LOW > __fdividef(200.f, c) && c < 1e8f;
        }
        // 0 * (-inf) must not get into w: a limit on t costs an instruction per logit, one on the packed logits half of one, and
        // serves where what it turns a logit into is zero too (of fp32 there is one per word: nothing is gained)
        if constexpr (!ENTROPY) {
            sum<T, U, false, false, false>(r, c, c1);
        } else if constexpr (Elem<T>::N == 8) {
            if (far) sum<T, U, false, true, false>(r, c, c1);
            else sum<T, U, false, false, true>(r, c, c1);
        } else {
            sum<T, U, false, false, true>(r, c, c1);
        }
        if (!tried) enter(c, c1);
    }
    // false, and nothing added, where a try has run over
    template <typename T, int U, bool TRY, bool LIMIT_X, bool LIMIT_T>
    __device__ __forceinline__ bool sum(const uint4 (&r)[U], float c, float c1) {
        constexpr int N = Elem<T>::N;
        const float base = TRY ? n : m == -INFINITY ? 0.f : m;
        const unsigned long long nb = pair(-base, -base), nb1 = pair(-n1, -n1), cc = pair(c, c), cc1 = pair(c1, c1);
        unsigned long long s2 = 0, w2 = 0, s12 = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4 v = r[u];
            if constexpr (LIMIT_X) {
                constexpr uint32_t low = Elem<T>::LOW2;
                v = make_uint4(Elem<T>::max2(v.x, low), Elem<T>::max2(v.y, low), Elem<T>::max2(v.z, low), Elem<T>::max2(v.w, low));
            }
            float f[N];
            Elem<T>::unpack(v, f);
            unsigned long long sv = 0, wv = 0;          // of the vector
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const unsigned long long x = pair(f[e], f[e + 1]), d = TRY ? x : add2(x, nb);
                float2 t = halves(TRY ? fma2(x, cc, nb) : mul2(d, cc));
                if (LIMIT_T) {
                    t.x = max_nan(t.x, T_MIN);
                    t.y = max_nan(t.y, T_MIN);
                }
                const unsigned long long q = pair(exp2_approx(t.x), exp2_approx(t.y));
                sv = e == 0 ? q : add2(sv, q);
                if (ENTROPY) wv = e == 0 ? mul2(q, pair(t.x, t.y)) : fma2(q, pair(t.x, t.y), wv);
                if (ONE == SQUARE) s12 = fma2(q, q, s12);
                if (ONE == OWN) {
                    const float2 t1 = halves(TRY ? fma2(x, cc1, nb1) : mul2(d, cc1));
                    s12 = add2(s12, pair(exp2_approx(t1.x), exp2_approx(t1.y)));
                }
            }
            s2 = u == 0 ? sv : add2(s2, sv);
            if (ENTROPY) w2 = u == 0 ? wv : add2(w2, wv);
        }
        const float2 a = halves(s2), b = halves(w2), a1 = halves(s12);
        const float ds = a.x + a.y, dw = b.x + b.y, ds1 = a1.x + a1.y;
        if (TRY && !(ds < TRY_BELOW && (!ENTROPY || fabsf(dw) < INFINITY) && (!ONE || ds1 < TRY_BELOW))) return false;
        if (ONE) s1 += ds1;
        if (!ENTROPY) {
            s += ds;
            return true;
        }
        // compensated, both at once
        const unsigned long long minus = pair(-1.f, -1.f), old = pair(s, w), y = fma2(pair(s_lost, w_lost), minus, pair(ds, dw));
        const unsigned long long sum = add2(old, y), lost = fma2(y, minus, fma2(old, minus, sum));
        const float2 now = halves(sum), gone = halves(lost);
        s = now.x;
        s_lost = gone.x;
        w = now.y;
        w_lost = gone.y;
        return true;
    }
};
// The CTA's sums, relative to its largest base, in every thread (`red`: 4 * WARPS floats).  all_ok: a thread's answer becomes the
// CTA's.
struct Sums {
    float m;
    double s, w, s1;
};
template <bool ENTROPY, AtOne ONE>
__device__ __forceinline__ Sums join_block(Running<ENTROPY, ONE> r, float c, float c1, float* red, bool* all_ok = nullptr) {
    if (ENTROPY) r.settle(c);
    else r.leave(c, c1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[warp] = m;
    if (all_ok != nullptr) *all_ok = __syncthreads_and(*all_ok);
    else __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m = max_nan(m, red[i]);
    if (!(m <= r.m)) r.raise(m, c, c1);
    const float s = warp_sum(r.s - r.s_lost), w = ENTROPY ? warp_sum(r.w - r.w_lost) : 0.f, s1 = ONE ? warp_sum(r.s1) : 0.f;
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
        if (ONE) t.s1 += red[3 * WARPS + i];
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

constexpr int BINS = 256;               // eight bits of a key
struct Selection {
    unsigned long long cand[MAX_CANDIDATES];
    unsigned long long best[MAX_K];
    uint4 stash[4][THREADS];                // vectors that a thread has read again
    unsigned short chosen[(SEGMENTS + 1) * THREADS];
    int bin[BINS];
    uint32_t hi[WARPS], lo[WARPS];
    float reach;
    int pick, above, through, crowded;
    int groups, count, scan[WARPS];
};

// The first k of the n candidates, in order, into `best`; returns how many there are.  All threads.
__device__ __forceinline__ int order_candidates(Selection& sel, int n, int k) {
    const int tid = threadIdx.x;
    if (n <= THREADS) {             // the place of a candidate is the number of those ahead of it: some lanes count for each
        const int shift = n <= THREADS / 8 ? 3 : n <= THREADS / 4 ? 2 : n <= THREADS / 2 ? 1 : 0, lanes = 1 << shift;
        const int at = tid >> shift, part = tid & (lanes - 1);
        const unsigned long long mine = at < n ? sel.cand[at] : 0;
        int ahead = 0;
#pragma unroll 4
        for (int i = part; i < n; i += lanes) ahead += sel.cand[i] > mine;
        for (int o = 1; o < lanes; o *= 2) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        if (part == 0 && at < n && ahead < k) sel.best[ahead] = mine;
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
// (What is out of line makes its slice anew: one passed by reference would live in memory all the while.)
template <typename T>
__device__ __noinline__ int select_by_passes(Selection& sel, const T* row, int V, int rank, int splits, int k) {
    constexpr int N = Elem<T>::N;
    const Slice<T> sl(row, V, rank, splits);
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

// The bin in which the need-th from above falls (sel.pick, -1 if there are fewer), and how many are above it.  First warp.
__device__ __forceinline__ void pick_bin(Selection& sel, int need) {
    constexpr int PER = BINS / 32;
    const int lane = threadIdx.x & 31;
    int n[PER], mine = 0;                               // lane 0 has the uppermost bins
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += n[i] = sel.bin[BINS - 1 - (lane * PER + i)];
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int above = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += above;
    }
    const uint32_t enough = __ballot_sync(0xffffffffu, upto >= need);
    if (enough == 0) {
        if (lane == 0) sel.pick = -1;
    } else if (lane == __ffs(enough) - 1) {
        int at = BINS, have = upto - mine, above = have;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (have < need) {
                above = have;
                have += n[i];
                at = BINS - 1 - (lane * PER + i);
            }
        sel.pick = at;
        sel.above = above;
        sel.through = have;
    }
}

// A value that at least k of the threads' largest values (two per thread) reach and hardly more do, into sel.reach: the edge of the
// bin of a histogram in which the k-th falls.  Where too many fall into it (values of masked vocabularies or outliers stretch the
// bins, values are equal) the k-th is found by the bits of its key, eight at a time.  NaN, which compares as reached, where there
// are fewer than k.
__device__ __forceinline__ void find_reach(Selection& sel, const float (&largest)[2], int k) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool some[2] = {!(largest[0] == -INFINITY), !(largest[1] == -INFINITY)};      // (no vectors, or nothing but -inf: not counted)
    const uint32_t key[2] = {key_of(largest[0]), key_of(largest[1])};
    const uint32_t hi = __reduce_max_sync(0xffffffffu, max(key[0], key[1]));
    const uint32_t lo = __reduce_min_sync(0xffffffffu, min(some[0] ? key[0] : 0xffffffffu, some[1] ? key[1] : 0xffffffffu));
    if (lane == 0) {
        sel.hi[warp] = hi;
        sel.lo[warp] = lo;
    }
    for (int i = tid; i < BINS; i += THREADS) sel.bin[i] = 0;
    __syncthreads();
    uint32_t top = 0, bottom = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        top = max(top, sel.hi[i]);
        bottom = min(bottom, sel.lo[i]);
    }
    const float from = value_of(bottom), scale = __fdividef(BINS - 0.01f, value_of(top) - from);    // (0 or NaN: one bin)
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (some[h]) atomicAdd(&sel.bin[min(BINS - 1, max(0, static_cast<int>((largest[h] - from) * scale)))], 1);
    __syncthreads();
    if (warp == 0) {
        pick_bin(sel, k);
        __syncwarp();
        if (lane == 0) {
            // below the bin's edge by more than the roundings of where its values are
            const float edge = from + static_cast<float>(sel.pick) / scale - (fabsf(from) + fabsf(value_of(top))) * 2e-6f;
            sel.reach = sel.pick < 0 ? __int_as_float(0x7fffffff) : edge;
            sel.crowded = sel.pick >= 0 && (sel.through > 2 * k + 64 || edge != edge);
            sel.groups = sel.count = 0;
        }
    }
    __syncthreads();
    if (sel.crowded) {
        uint32_t prefix = 0;
        int need = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < BINS; i += THREADS) sel.bin[i] = 0;
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (some[h] && (shift == 24 || key[h] >> (shift + 8) == prefix)) atomicAdd(&sel.bin[key[h] >> shift & 255], 1);
            __syncthreads();
            if (warp == 0) pick_bin(sel, need);
            __syncthreads();
            prefix = prefix << 8 | static_cast<uint32_t>(sel.pick);
            need -= sel.above;
        }
        if (tid == 0) sel.reach = value_of(prefix);
        __syncthreads();
    }
}

// The k best of a slice, in order, into sel.best; returns how many the slice has.  The stream has left each thread's largest
// value and those of its segments (`group`).  What reaches the k-th largest of the threads' values are k values at least and
// hardly more (where values come in no order 1.4 k for k = 64, 1.3 k for 100, 1.4 k for 128), so only the segments that do are
// read again.  Few instructions matter more than few reads: the other CTAs of the SM stream meanwhile, and a warp gets every
// sixth slot.
// Slices of fewer than k threads with vectors (a warp takes 128 vectors before the next has any) have no such value: all of
// theirs are candidates, and from 1025 on they go through select_by_passes.  4096 x 2000 bf16, best 64 (63 threads): 92 us, best 80
// 367, best 20 31; one row of 8200 in 8 slices, best 64 or more: 72 to 80 us, best 20 14.
template <typename T>
__device__ __noinline__ int select_best(Selection& sel, const float* group, const T* row, int V, int rank, int splits, int k,
                                        float largest, int segment_shift) {
    constexpr int N = Elem<T>::N, AHEAD = 4;
    const Slice<T> sl(row, V, rank, splits);
    const int tid = threadIdx.x;
    // Nearly as many as there are threads: the smallest of their largest values say little (the k-th of 128 is reached by 700
    // values for k = 128, and by more than there is room for in every twentieth row).  Odd and even segments by themselves make
    // twice as many.  4096 x 128256 bf16 with one value per thread and with two: best 80 224 and 210 us, 100 245 and 226, 128 3370
    // and 240.
    float halves[2] = {largest, -INFINITY};
    if (k > THREADS / 2) {
        halves[0] = -INFINITY;
#pragma unroll
        for (int i = 0; i < SEGMENTS + 1; ++i) halves[i & 1] = max_nan(halves[i & 1], group[i * THREADS + tid]);
    }
    find_reach(sel, halves, k);
    const float reach = sel.reach;
    if (!(largest < reach)) {
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < SEGMENTS + 1; ++i) mask |= (group[i * THREADS + tid] < reach ? 0u : 1u) << i;
        for (int at = atomicAdd(&sel.groups, __popc(mask)); mask != 0; mask &= mask - 1)
            sel.chosen[at++] = static_cast<unsigned short>((__ffs(mask) - 1) * THREADS + tid);
    }
    __syncthreads();
    const int shift = segment_shift + 2, items = sel.groups << shift;       // a segment has 4 vectors of each of its steps
    static_assert(UNROLL == 4, "");
    for (int i0 = tid; i0 < items; i0 += AHEAD * THREADS) {
        uint4 v[AHEAD];
        int at[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int i = i0 + a * THREADS;
            at[a] = -1;
            if (i >= items) continue;
            const int chosen = sel.chosen[i >> shift], q = i & ((1 << shift) - 1), segment = chosen / THREADS, t = chosen % THREADS;
            if (segment == SEGMENTS) {                  // the parts at the row's ends
                if (q == 0 && t == 0 && sl.head) at[a] = 0;
                if (q == 0 && t == 1 && sl.tail) at[a] = sl.nv - 1;
            } else {
                const int j = sl.full0 + ((segment << segment_shift) + q / UNROLL) * (THREADS * UNROLL) + (t >> 5) * WARP_STEP +
                              q % UNROLL * 32 + (t & 31);
                if (j < sl.full1) at[a] = j;
            }
            if (at[a] >= 0) v[a] = sl.load_any(at[a]);
        }
        uint32_t hits = 0;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (at[a] < 0) continue;
            float f[N];
            Elem<T>::unpack(v[a], f);
#pragma unroll
            for (int e = 0; e < N; ++e) hits |= (f[e] < reach ? 0u : 1u) << (N * a + e);
        }
        if (hits != 0) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) sel.stash[a][tid] = v[a];
            int to = atomicAdd(&sel.count, __popc(hits));
            for (; hits != 0; hits &= hits - 1) {
                const int b = __ffs(hits) - 1, a = b / N;
                const int id = sl.index(a == 0 ? at[0] : a == 1 ? at[1] : a == 2 ? at[2] : at[3], b % N);
                const float x = Elem<T>::f(get<T>(sel.stash[a][tid], b % N));
                // (0 for the places of a part that are not the row's: they come last)
                if (to < MAX_CANDIDATES) sel.cand[to] = id >= 0 && id < sl.V ? candidate(key_of(x), id) : 0ull;
                ++to;
            }
        }
    }
    __syncthreads();
    int n = sel.count;
    if (n > MAX_CANDIDATES) n = select_by_passes<T>(sel, row, V, rank, splits, k);
    __syncthreads();
    return min(order_candidates(sel, n, k), sl.size());
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

// Six CTAs of four warps per SM with 80 registers: with more and fewer registers the tried steps take more instructions
// (4094 x 128256 bf16, sustained: 183 us, 189 with seven; three CTAs of eight warps: 190, and 52 instead of 27 at 8192 x 2048,
// where what surrounds a row's stream counts).
template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 6) token_logprobs_kernel(const __grid_constant__ ScoreArgs p) {
    __shared__ float red[4 * WARPS];
    __shared__ uint64_t ring_bars[WARPS * RING_STAGES];
    __shared__ float part_m;
    __shared__ double part_s, part_w, row_log_s;
    __shared__ int part_n;
    extern __shared__ __align__(128) uint8_t vocab_smem[];      // the ring, and once it is empty the selection
    __shared__ float group_[TOP ? (SEGMENTS + 1) * THREADS : 1];
    Selection& sel = *reinterpret_cast<Selection*>(vocab_smem);
    float* group = group_;
    const int tid = threadIdx.x;
    const unsigned splits = p.splits, row_index = splits == 1 ? blockIdx.x : blockIdx.x / splits;
    const long long r = row_index;
    const int rank = blockIdx.x - row_index * splits;
    const T* row = p.rows.row<T>(r);
    const Slice<T> sl(row, p.rows.V, rank, p.splits);
    const float c = static_cast<float>(p.inv_temperature * 1.4426950408889634);

    Ring<T> ring(sl, vocab_smem, ring_bars);
    long long tok = 0;              // of the thread that finishes the row
    float x_tok = 0.f;
    if (p.tokens != nullptr && rank == 0 && tid == THREADS - 1) {
        tok = p.tokens[r];
        if (tok >= 0 && tok < p.rows.V) x_tok = Elem<T>::f(row[tok]);
    }
    Running<true, NONE> run;
    const int steps = sl.steps();
    int segment_shift = 0;              // a segment has 2^segment_shift steps
    while (steps > SEGMENTS << segment_shift) ++segment_shift;
    if constexpr (TOP)
        for (int i = 0; i < SEGMENTS + 1; ++i) group[i * THREADS + tid] = -INFINITY;
    float largest = -INFINITY;          // of the segment
    float mine = -INFINITY;             // this thread's
    int left = 1 << segment_shift, segment = 0;
    ring.stream([](int, uint32_t) {}, [&](int step, uint4 (&v)[UNROLL], bool whole) {
        if constexpr (!TOP) {
            run.template add<T>(v, whole, [&] { return max_of<T>(v); }, c, 0.f);
        } else {
            const float m = max_of<T>(v);
            run.template add<T>(v, whole, [&] { return m; }, c, 0.f);
            largest = max_nan(largest, m);
            if (--left == 0 || step == ring.steps - 1) {
                group[segment * THREADS + tid] = largest;
                mine = max_nan(mine, largest);
                ++segment;
                left = 1 << segment_shift;
                largest = -INFINITY;
            }
        }
    });
    if ((tid == 0 && sl.head) || (tid == 1 && sl.tail)) {
        const uint4 v[1] = {sl.load_part(tid == 0 ? 0 : sl.nv - 1)};
        const float m = max_of<T>(v);
        run.template add<T>(v, false, [&] { return m; }, c, 0.f);
        if constexpr (TOP) {
            group[SEGMENTS * THREADS + tid] = m;
            mine = max_nan(mine, m);
        }
    }
    bool arrived = ring.ok;             // if not, the ring's memory may still be written to and serves nothing else
    Sums sum = join_block(run, c, 0.f, red, TOP ? &arrived : nullptr);
    // the row's last values: one thread of the last warp, while the others select
    auto finish = [&] {
        const double log_s = log(sum.s), entropy = log_s - sum.w / sum.s * LN2;
        if (p.tokens != nullptr) {
            float lp = 0.f;
            if (tok != p.ignore_index)
                lp = tok >= 0 && tok < p.rows.V ? static_cast<float>((static_cast<double>(x_tok) - sum.m) * p.inv_temperature - log_s)
                                                : __int_as_float(0x7fffffff);
            p.logprobs[r] = lp;
        }
        p.entropy[r] = static_cast<float>(entropy);
        if (p.stats != nullptr)
            *reinterpret_cast<float4*>(p.stats + 4 * r) = make_float4(sum.m, static_cast<float>(sum.s), static_cast<float>(entropy),
                                                                     static_cast<float>(log_s));
        row_log_s = log_s;
    };
    if (p.splits == 1 && tid == THREADS - 1) finish();
    int n = 0;
    if constexpr (TOP)
        if (arrived) n = select_best<T>(sel, group, row, p.rows.V, rank, p.splits, p.k, mine, segment_shift);

    if (p.splits > 1) {
        if (tid == 0) {
            part_m = sum.m;
            part_s = sum.s;
            part_w = sum.w;
            part_n = n;
        }
        cluster_sync();
        if (rank == 0) {
            // every warp joins the parts, a lane for each
            const int lane = tid & 31;
            const bool there = lane < p.splits;
            const float mq = there ? ld_peer(&part_m, lane) : -INFINITY;
            const int nq = there ? ld_peer(&part_n, lane) : 0;
            double s = there ? ld_peer(&part_s, lane) : 0.0, w = there ? ld_peer(&part_w, lane) : 0.0;
            float m = mq;
#pragma unroll
            for (int o = MAX_SPLITS / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            m = __shfl_sync(0xffffffffu, m, 0);
            const float t = mq == m ? 0.f : max_nan((mq - m) * c, T_MIN), f = there ? exp2f(t) : 0.f;
            w = (w + s * t) * f;
            s = s * f;
#pragma unroll
            for (int o = MAX_SPLITS / 2; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                w += __shfl_xor_sync(0xffffffffu, w, o);
            }
            sum = Sums{m, __shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, w, 0), 0.0};
            if (tid == THREADS - 1) finish();
            if constexpr (TOP) {
                if (arrived) {
                    int base = 0;
                    __syncthreads();
                    for (int q = 0; q < p.splits; ++q) {
                        const int nb = __shfl_sync(0xffffffffu, nq, q);
                        for (int i = tid; i < nb; i += THREADS) sel.cand[base + i] = ld_peer(&sel.best[i], q);
                        base += nb;
                    }
                    __syncthreads();
                    n = order_candidates(sel, base, p.k);
                }
            }
        }
    }
    if constexpr (TOP) {
        if (rank == 0) {
            __syncthreads();
            if (tid < n) {
                const unsigned long long b = sel.best[tid];
                p.top_ids[r * p.k + tid] = index_of(b);
                p.top_logprobs[r * p.k + tid] = static_cast<float>(
                    (static_cast<double>(value_of(static_cast<uint32_t>(b >> 32))) - sum.m) * p.inv_temperature - row_log_s);
            } else if (tid < p.k) {     // (only where something has not arrived: an id that may be used as an index)
                p.top_ids[r * p.k + tid] = 0;
                p.top_logprobs[r * p.k + tid] = __int_as_float(0x7fffffff);
            }
        }
    }
    if (p.splits > 1) cluster_sync();   // the leader has read this CTA's part
}

// ------------------------------------------------------------------ gradients
// dx_j = coefficient of the row times the row's exponentials, and other values at single tokens, which overwrite what the
// stream has stored once the CTA has passed a barrier.  A CTA takes some steps of one row: nothing depends on the other
// CTAs.
template <typename T>
struct GradSlice {
    static constexpr int N = Elem<T>::N;
    const T* x;
    T* out;
    int V, before, begin, end;      // vectors are those of the output; [begin, end) are this CTA's
    int full0, full1;               // whole ones of the row
    bool same;                      // rows of both tensors start at the same place of a vector

    __device__ __forceinline__ GradSlice(const T* x_, T* out_, int V_, int chunk, int steps) : x(x_), out(out_), V(V_) {
        before = static_cast<int>((reinterpret_cast<uintptr_t>(out_) & 15) / sizeof(T));
        same = before == static_cast<int>((reinterpret_cast<uintptr_t>(x_) & 15) / sizeof(T));
        const int nv = (before + V + N - 1) / N;
        begin = min(nv, chunk * steps * (THREADS * UNROLL));
        end = min(nv, begin + steps * (THREADS * UNROLL));
        full0 = before > 0 ? 1 : 0;
        full1 = (before + V) / N;
    }
    __device__ __forceinline__ bool has(int id) const {
        const int j = (id + before) / N;
        return id >= 0 && id < V && j >= begin && j < end;
    }
    __device__ __forceinline__ bool smooth(int j) const {       // a step that begins at vector j has whole ones only
        return j >= full0 && j + THREADS * UNROLL <= min(end, full1);
    }
    __device__ __forceinline__ const T* at(const T* p, int j) const { return p - before + static_cast<long long>(j) * N; }
    __device__ __forceinline__ void load_step(int j0, uint4 (&v)[UNROLL]) const {
        const int j = j0 + threadIdx.x;
        if (same && smooth(j0)) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w) : "l"(at(x, j + u * THREADS)));
        } else {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int q = j + u * THREADS;
                if (q >= end) continue;
                if (same && q >= full0 && q < full1) {
                    v[u] = *reinterpret_cast<const uint4*>(at(x, q));
                    continue;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int k = q * N + i - before;
                    put(v[u], i, k >= 0 && k < V ? x[k] : Elem<T>::from(0.f));
                }
            }
        }
    }
    __device__ __forceinline__ void store_step(int j0, const uint4 (&v)[UNROLL]) const {
        const int j = j0 + threadIdx.x;
        if (smooth(j0)) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) *reinterpret_cast<uint4*>(const_cast<T*>(at(out, j + u * THREADS))) = v[u];
        } else {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int q = j + u * THREADS;
                if (q >= end) continue;
                if (q >= full0 && q < full1) {
                    *reinterpret_cast<uint4*>(const_cast<T*>(at(out, q))) = v[u];
                    continue;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int k = q * N + i - before;
                    if (k >= 0 && k < V) out[k] = get<T>(v[u], i);
                }
            }
        }
    }
    // out_j = f(x_j), two at a time; the next step's loads on their way
    template <typename F>
    __device__ __forceinline__ void map(F&& f) const {
        uint4 v[UNROLL], next[UNROLL];
        if (begin < end) load_step(begin, v);
        for (int j = begin; j < end; j += THREADS * UNROLL) {
            if (j + THREADS * UNROLL < end) load_step(j + THREADS * UNROLL, next);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                float e[N];
                Elem<T>::unpack(v[u], e);
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const float2 y = halves(f(pair(e[i], e[i + 1])));
                    e[i] = y.x;
                    e[i + 1] = y.y;
                }
                v[u] = Elem<T>::pack(e);
            }
            store_step(j, v);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) v[u] = next[u];
        }
    }
    __device__ __forceinline__ void zero() const {
        const uint4 z[UNROLL] = {};
        for (int j = begin; j < end; j += THREADS * UNROLL) store_step(j, z);
    }
};

struct ScoreGradArgs {
    Rows rows;
    void* grad;                     // [rows][V], dense
    const long long* tokens;
    long long ignore_index;
    float inv_temperature;
    int k, chunks, steps;           // CTAs per row, and steps of a CTA
    const float* stats;
    const long long* top_ids;
    const float *d_logprobs, *d_entropy, *d_top;        // any may be null
};

// dx_j = (1 / temperature) (d_tok (1[tok = j] - p_j) - d_ent p_j (log p_j + H) + sum_i d_top_i (1[id_i = j] - p_j))
template <typename T>
__global__ void __launch_bounds__(THREADS, 8) token_logprobs_grad_kernel(const __grid_constant__ ScoreGradArgs p) {
    __shared__ float red[32];
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / static_cast<unsigned>(p.chunks);
    const int V = p.rows.V;
    T* out = static_cast<T*>(p.grad) + r * V;
    const GradSlice<T> g(p.rows.row<T>(r), out, V, blockIdx.x % static_cast<unsigned>(p.chunks), p.steps);
    const float4 st = *reinterpret_cast<const float4*>(p.stats + 4 * r);
    const float m = st.x, inv_s = 1.f / st.y, c = p.inv_temperature * LOG2E;
    int tok = -1;
    float d_tok = 0.f;
    if (p.d_logprobs != nullptr) {
        const long long i = p.tokens[r];
        if (i != p.ignore_index && i >= 0 && i < V) {
            tok = static_cast<int>(i);
            d_tok = p.d_logprobs[r] * p.inv_temperature;
        }
    }
    const float d_ent = p.d_entropy != nullptr ? p.d_entropy[r] * p.inv_temperature : 0.f;
    int id = -1;
    float d_id = 0.f, d_all = d_tok;
    if (p.d_top != nullptr) {
        if (tid < p.k) {
            id = static_cast<int>(p.top_ids[r * p.k + tid]);
            d_id = p.d_top[r * p.k + tid] * p.inv_temperature;
        }
        d_all += block_sum(d_id, red);
    }
    // p_j (a + b log p_j), log p_j = ln2 t_j - log S
    const float a = -(d_all + d_ent * st.z), b = -d_ent;
    const float a2 = inv_s * (a - b * st.w), b2 = inv_s * b * static_cast<float>(LN2);
    const unsigned long long nm = pair(-m, -m), cc = pair(c, c), aa = pair(a2, a2), bb = pair(b2, b2);
    auto value = [&](unsigned long long x) {
        float2 t = halves(mul2(add2(x, nm), cc));
        t.x = max_nan(t.x, T_MIN);
        t.y = max_nan(t.y, T_MIN);
        return mul2(pair(exp2_approx(t.x), exp2_approx(t.y)), fma2(bb, pair(t.x, t.y), aa));
    };
    auto value_at = [&](int i) {
        const float x = Elem<T>::f(g.x[i]);
        return halves(value(pair(x, x))).x;
    };
    g.map(value);
    const bool here = g.has(id), met = here && id == tok;
    const bool taken = __syncthreads_or(met);
    if (here) out[id] = Elem<T>::from(value_at(id) + d_id + (met ? d_tok : 0.f));
    if (tid == 0 && !taken && g.has(tok)) out[tok] = Elem<T>::from(value_at(tok) + d_tok);
}

// ------------------------------------------------------------------ distillation from a teacher's best tokens
// q: the teacher's listed tokens, and with a tail one bucket for all others, q_r = 1 - sum q.  p: the student, p_r the sum
// over the tokens that are not listed.  KL(q || p), or with forward_kl KL(p || q), over the buckets.  p_r is summed as
// such and not as 1 - sum p, which would leave nothing of a small rest: the listed tokens are bits of a map in shared memory,
// a word for a lane's vectors of a step, and the stream writes minus infinity over them before it reads a stage.
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
    float* stats;                   // [rows][12]
};
// stats, for the gradient.  Tokens that are not listed: base m_r of their exponentials, what these are multiplied by for the
// divergence and for the cross entropy, and 2 if the row has a divergence, 1 if it has a label only, 0 if neither.  Listed ones:
// base m, 1 / S, log S, sum q + q_r (with forward_kl the divergence); what is taken from the teacher's values to make them log
// probabilities (in two parts), 1 / S at temperature one.  Two bases, since all that is not listed may be less likely than fp32 can say.

struct DistillPart {        // of a CTA
    float m, mr;            // largest of its bases, and that of the tokens that are not listed
    int n;                  // listed tokens that count
    double rest, rest1;     // sums of exponentials relative to mr: not listed, the same at temperature one
    double top, top1;       // relative to m: listed
    double q, qx;           // sum of the teacher's weights u, sum of u (its log - x / temperature)
    double px;              // forward_kl: sum of listed exponentials times (x / temperature - teacher's log)
};

// As above (8192 x 128256 bf16: 350 us, 375 with eight CTAs of fewer registers; 2047 x 50257: 46 and 44).
template <typename T, AtOne ONE>
__global__ void __launch_bounds__(THREADS, 6) topk_distillation_kernel(const __grid_constant__ DistillArgs p) {
    constexpr int N = Elem<T>::N;
    extern __shared__ __align__(128) uint8_t vocab_smem[];  // the ring, then the map
    uint32_t* listed = reinterpret_cast<uint32_t*>(vocab_smem + RING_BYTES);
    __shared__ float red[4 * WARPS];
    __shared__ uint64_t ring_bars[WARPS * RING_STAGES];
    __shared__ int id_of[MAX_K];
    __shared__ DistillPart part;
    __shared__ double part_of[MAX_K / 32][4];
    __shared__ float list_max[2][MAX_K / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned splits = p.splits, row_index = splits == 1 ? blockIdx.x : blockIdx.x / splits;
    const long long r = row_index;
    const int rank = blockIdx.x - row_index * splits;
    const int V = p.rows.V;
    const T* row = p.rows.row<T>(r);
    const Slice<T> sl(row, V, rank, p.splits);
    const float c = static_cast<float>(p.inv_temperature * 1.4426950408889634);

    Ring<T> ring(sl, vocab_smem, ring_bars);
    // the list: entries that count are in the vocabulary, have a finite or NaN value, and come first of their token
    static_assert(UNROLL == 4, "a word of the map has a lane's vectors of a step");
    const int words = (sl.full1 - sl.full0 + WARP_STEP - 1) / WARP_STEP * 32;       // and one each for the parts at the ends
    for (int i = tid; i < words + 2; i += THREADS) listed[i] = 0;
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
    if (!any && !labelled) {            // nothing is asked of this row: it is not read, but for what the ring has under way
        ring.drain();
        if (rank == 0) {
            if (tid < p.k) p.entries[r * p.k + tid] = -1;
            if (tid == 0) {
                p.kl[r] = 0.f;
                if (p.nll != nullptr) p.nll[r] = 0.f;
            }
            if (tid < 12) p.stats[12 * r + tid] = 0.f;
        }
        return;                         // (all CTAs of the cluster alike)
    }
    const bool mine = id >= 0 && sl.has(id);
    bool again = false;
    if (mine) {
        const int j = (id + sl.before) / N, q = j - sl.full0;
        const int word = sl.whole(j) ? q / WARP_STEP * 32 + q % 32 : words + (j == 0 ? 0 : 1);
        const int bit = (sl.whole(j) ? q % WARP_STEP / 32 * 8 : 0) + (id + sl.before) % N;
        again = atomicOr(&listed[word], 1u << bit) >> bit & 1u;
    }
    // Only an id's first entry counts, also for the largest value, which is of the whole list and asked for without a tail: this
    // CTA's map says nothing of ids in the others.
    bool first = id >= 0;
    if (__syncthreads_or(again) || (p.splits > 1 && !p.tail))
        if (first)
            for (int i = 0; i < tid; ++i) first &= id_of[i] != id;
    const bool counts = mine && first;
    if (tid < p.k && (mine || (rank == 0 && id < 0))) p.entries[r * p.k + tid] = counts ? id : -1;
    const float x = counts ? Elem<T>::f(row[id]) : -INFINITY;
    const float x_label = rank == 0 && tid == 0 && labelled && label >= 0 && label < V ? Elem<T>::f(row[label]) : 0.f;

    Running<false, ONE> run;
    ring.stream(
        [&](int step, uint32_t address) {
            uint32_t bits = listed[(step * WARPS + warp) * 32 + lane];
            if (bits != 0) {        // a lane's own vectors, which it reads next
                for (; bits != 0; bits &= bits - 1) {
                    const int b = __ffs(bits) - 1;
                    const uint32_t at = address + b / 8 * 512 + b % 8 * static_cast<int>(sizeof(T));
                    if constexpr (sizeof(T) == 2)
                        asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(Elem<T>::NEG_INF & 0xffffu)) : "memory");
                    else
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(Elem<T>::NEG_INF) : "memory");
                }
            }
        },
        [&](int, uint4 (&v)[UNROLL], bool whole) {
            run.template add<T>(v, whole, [&] { return max_of<T>(v); }, c, LOG2E);
        });
    if ((tid == 0 && sl.head) || (tid == 1 && sl.tail)) {
        uint4 v[1] = {sl.load_part(tid == 0 ? 0 : sl.nv - 1)};
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (listed[words + tid] >> i & 1u) put(v[0], i, Elem<T>::from(-INFINITY));
        run.template add<T>(v, false, [&] { return max_of<T>(v); }, c, LOG2E);
    }
    Sums sum = join_block(run, c, LOG2E, red);

    // the listed tokens, in 64 bits.  Weights without a tail are relative to the largest value of the list.
    float m = max_nan(x, -INFINITY), ref = first ? lq : -INFINITY;
    static_assert(MAX_K == THREADS, "every warp has a part of the list");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        ref = max_nan(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    }
    if (lane == 0) {
        list_max[0][warp] = m;
        list_max[1][warp] = ref;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MAX_K / 32; ++i) {
        m = max_nan(m, list_max[0][i]);
        ref = max_nan(ref, list_max[1][i]);
    }
    m = max_nan(m, sum.m);
    if (p.tail || ref == -INFINITY) ref = 0.f;
    double e[4] = {0, 0, 0, 0};     // listed exponentials, at temperature one, weights, products
    if (counts) {
        const double d = static_cast<double>(x) - m, y = static_cast<double>(x) * p.inv_temperature;
        e[0] = x == -INFINITY ? 0.0 : exp(d * p.inv_temperature);
        if (ONE) e[1] = x == -INFINITY ? 0.0 : exp(d);
        e[2] = exp(static_cast<double>(lq) - ref);
        if (p.forward_kl) e[3] = e[0] == 0.0 ? 0.0 : e[0] * (y - lq);
        else e[3] = e[2] == 0.0 ? 0.0 : e[2] * (static_cast<double>(lq) - ref - y);
    }
    if (p.k > 32 * warp) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (ONE || q != 1)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) e[q] += __shfl_xor_sync(0xffffffffu, e[q], o);
    }
    if (lane == 0)
        for (int q = 0; q < 4; ++q) part_of[warp][q] = e[q];
    const int n = __syncthreads_count(counts);
    if (warp > 0 && p.splits == 1) return;
    if (tid == 0) {
        double e[4];
        for (int q = 0; q < 4; ++q) {
            e[q] = 0;
            for (int i = 0; i < MAX_K / 32; ++i) e[q] += part_of[i][q];
        }
        part = DistillPart{m, sum.m, n, sum.s, sum.s1, e[0], e[1], e[2], p.forward_kl ? 0.0 : e[3], p.forward_kl ? e[3] : 0.0};
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync();
    if (rank == 0 && warp == 0) {
        DistillPart all = part;
        if (p.splits > 1) {             // a lane for each part
            const bool there = lane < p.splits;
            const DistillPart* q = &part;
            all.m = there ? ld_peer(&q->m, lane) : -INFINITY;
            all.mr = there ? ld_peer(&q->mr, lane) : -INFINITY;
            all.n = there ? ld_peer(&q->n, lane) : 0;
            all.rest = there ? ld_peer(&q->rest, lane) : 0;
            all.top = there ? ld_peer(&q->top, lane) : 0;
            all.rest1 = there && ONE ? ld_peer(&q->rest1, lane) : 0;
            all.top1 = there && ONE ? ld_peer(&q->top1, lane) : 0;
            all.q = there ? ld_peer(&q->q, lane) : 0;
            all.qx = there ? ld_peer(&q->qx, lane) : 0;
            all.px = there ? ld_peer(&q->px, lane) : 0;
            float largest = all.m, largest_r = all.mr;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
                largest_r = max_nan(largest_r, __shfl_xor_sync(0xffffffffu, largest_r, o));
            }
            if (there && all.m != largest) {
                const double d = fmax(static_cast<double>(all.m) - largest, -1e30), f = exp(d * p.inv_temperature);
                all.top *= f;
                all.px *= f;
                if (ONE) all.top1 *= exp(d);
            }
            if (there && all.mr != largest_r) {
                const double d = fmax(static_cast<double>(all.mr) - largest_r, -1e30);
                all.rest *= exp(d * p.inv_temperature);
                if (ONE) all.rest1 *= exp(d);
            }
            all.m = largest;
            all.mr = largest_r;
            double* v[7] = {&all.rest, &all.top, &all.rest1, &all.top1, &all.q, &all.qx, &all.px};
#pragma unroll
            for (int o = MAX_SPLITS / 2; o > 0; o >>= 1) {
                all.n += __shfl_xor_sync(0xffffffffu, all.n, o);
#pragma unroll
                for (int i = 0; i < 7; ++i) *v[i] += __shfl_xor_sync(0xffffffffu, *v[i], o);
            }
        }
        // the logarithms, a lane for each, then one thread.  What is not listed stays in the logarithm: its probability may be
        // less than a double can say.
        const double down = all.rest > 0 ? static_cast<double>(all.mr) - all.m : all.rest == 0 ? 0.0 : all.rest;    // (or NaN)
        const double S = all.top + all.rest * exp(down * p.inv_temperature);
        const double S1 = ONE ? all.top1 + all.rest1 * exp(down) : S;
        double q_r = p.tail ? 1 - all.q : 0.0;
        if (q_r < NO_TAIL) q_r = 0;
        const double logs = log(lane == 0   ? S
                                : lane == 1 ? all.rest
                                : lane == 2 ? fmax(q_r, NO_TAIL)
                                : lane == 3 ? all.q
                                : lane == 4 ? S1
                                            : all.rest1);
        const double log_s = __shfl_sync(0xffffffffu, logs, 0), log_rest = __shfl_sync(0xffffffffu, logs, 1);
        const double log_q_r = __shfl_sync(0xffffffffu, logs, 2), log_q = __shfl_sync(0xffffffffu, logs, 3);
        const double log_s1 = __shfl_sync(0xffffffffu, logs, 4), log_rest1 = __shfl_sync(0xffffffffu, logs, 5);
        if (lane == 0) {
            const bool others = all.rest != 0;      // (NaN too)
            const double lse = all.m * p.inv_temperature + log_s, log_p_r = log_rest + down * p.inv_temperature - log_s;
            const double p_r = others ? exp(log_p_r) : 0.0;
            double kl = 0, factor = 0, fourth = 0, norm = 0;
            if (all.n > 0) {
                if (!p.forward_kl) {
                    if (p.tail) {
                        kl = all.qx + all.q * lse;
                        if (q_r > 0) kl += q_r * (log_q_r - log_p_r);
                        fourth = all.q + (others ? q_r : 0.0);
                    } else {
                        norm = ref + log_q;
                        kl = all.qx / all.q - log_q + lse;
                        fourth = 1;
                    }
                    factor = fourth * p_r - q_r;
                } else {
                    const double ratio = others ? log_p_r - log_q_r : 0.0;
                    kl = (all.px - all.top * lse) / S + p_r * ratio;
                    fourth = kl;
                    factor = p_r * (ratio - kl);
                }
            }
            p.kl[r] = static_cast<float>(kl);
            if (p.nll != nullptr)
                p.nll[r] = !labelled              ? 0.f
                           : label >= 0 && label < V ? static_cast<float>(log_s1 - (static_cast<double>(x_label) - all.m))
                                                     : __int_as_float(0x7fffffff);
            // The gradient's exponentials are relative to where their sums are about one (at both temperatures at least one), so
            // that the logarithms that it subtracts are small.
            double up = log_s / p.inv_temperature, up_r = log_rest / p.inv_temperature;
            if (ONE) {
                up = fmin(up, log_s1);
                up_r = fmin(up_r, log_rest1);
            }
            const float m2 = static_cast<float>(all.m + up), mr2 = others ? static_cast<float>(all.mr + up_r) : S > 0 ? 0.f : m2 - m2;
            const double moved = static_cast<double>(m2) - all.m, log_s2 = log_s - moved * p.inv_temperature;
            const double inv_rest = others ? exp((static_cast<double>(mr2) - all.mr) * p.inv_temperature - log_rest) : 0.0;
            const double of_nll = ONE ? (others ? exp(static_cast<double>(mr2) - all.m - log_s1) : 0.0) : p_r * inv_rest;
            float4* st = reinterpret_cast<float4*>(p.stats + 12 * r);
            st[0] = make_float4(mr2, static_cast<float>(factor * inv_rest), static_cast<float>(of_nll), all.n > 0 ? 2.f : 1.f);
            st[1] = make_float4(m2, static_cast<float>(exp(-log_s2)), static_cast<float>(log_s2), static_cast<float>(fourth));
            const float norm_hi = static_cast<float>(norm);     // (raw logits may have any offset)
            st[2] = make_float4(norm_hi, static_cast<float>(norm - norm_hi), static_cast<float>(exp(moved - log_s1)), 0.f);
        }
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
    int k, chunks, steps, forward_kl;
    const float* stats;
    const float *d_kl, *d_nll;      // either may be null
};

// Tokens that are not listed: p_j times the row's factor.  Listed ones: p_i (sum q + q_r) - q_i, with forward_kl
// p_i (log p_i - log q_i - KL).  Both over the temperature, and the cross entropy's p_j - 1[label = j] on top.
template <typename T, AtOne ONE>
__global__ void __launch_bounds__(THREADS, 8) topk_distillation_grad_kernel(const __grid_constant__ DistillGradArgs p) {
    const int tid = threadIdx.x;
    const long long r = blockIdx.x / static_cast<unsigned>(p.chunks);
    const int V = p.rows.V;
    T* out = static_cast<T*>(p.grad) + r * V;
    const GradSlice<T> g(p.rows.row<T>(r), out, V, blockIdx.x % static_cast<unsigned>(p.chunks), p.steps);
    const float4* st = reinterpret_cast<const float4*>(p.stats + 12 * r);
    const float4 others = st[0];
    if (others.w == 0.f) {          // no loss: not read, gradient zero
        g.zero();
        return;
    }
    const float c = p.inv_temperature * LOG2E;
    const float d_kl = p.d_kl != nullptr && others.w == 2.f ? p.d_kl[r] * p.inv_temperature : 0.f;
    int label = -1;
    float d_nll = 0.f;
    if (p.d_nll != nullptr) {
        const long long i = p.labels[r];
        if (i != p.ignore_index && i >= 0 && i < V) {
            label = static_cast<int>(i);
            d_nll = p.d_nll[r];
        }
    }
    const float a = d_kl * others.y + (ONE ? 0.f : d_nll * others.z), a1 = d_nll * others.z;
    const unsigned long long nm = pair(-others.x, -others.x), cc = pair(c, c), cc1 = pair(LOG2E, LOG2E), aa = pair(a, a);
    const unsigned long long aa1 = pair(a1, a1);
    auto value = [&](unsigned long long x) {        // (at listed tokens it may run over: they get theirs below)
        const unsigned long long d = add2(x, nm);
        const float2 t = halves(mul2(d, cc));
        const unsigned long long e = pair(exp2_approx(t.x), exp2_approx(t.y)), v = mul2(e, aa);
        if (ONE == NONE) return v;
        if (ONE == SQUARE) return fma2(mul2(e, e), aa1, v);
        const float2 t1 = halves(mul2(d, cc1));
        return fma2(pair(exp2_approx(t1.x), exp2_approx(t1.y)), aa1, v);
    };
    g.map(value);
    int id = -1;
    if (tid < p.k) id = p.entries[r * p.k + tid];
    const bool here = g.has(id), met = here && id == label;
    const bool taken = __syncthreads_or(met);
    if (here) {         // (fp32, and an exponential that is off by a step or two and one more for each nat)
        const float4 top = st[1], more = st[2];
        const float d = Elem<T>::f(g.x[id]) - top.x, t = d * c, e = exp2_approx(t) * top.y;
        const float lq = p.teacher[r * p.k + tid] - more.x - more.y;
        float v;
        if (p.forward_kl) v = e == 0.f ? 0.f : e * (t * static_cast<float>(LN2) - top.z - lq - top.w);
        else v = e * top.w - __expf(lq);
        v = v * d_kl + d_nll * (ONE ? exp2_approx(d * LOG2E) * more.z : e) - (met ? d_nll : 0.f);
        out[id] = Elem<T>::from(v);
    }
    if (tid == 0 && !taken && g.has(label)) {
        const float x = Elem<T>::f(g.x[label]);
        out[label] = Elem<T>::from(halves(value(pair(x, x))).x - d_nll);
    }
}

// ------------------------------------------------------------------ launches
// CTAs per row: as many as fit on the GPU at once (six per SM) for all rows, while each keeps about a vector for every other thread
// at least.  Forward kernels with two CTAs per row and with one, us:
//                        bf16, 128256 logits      fp32, 32000 logits       bf16, 32000 logits
//   rows                 223        333           223        333           223        333        444
//   scores               16.4 19.9  20.0 23.0      9.8 10.8  11.8 12.1      7.9  8.1   9.7  9.1  10.7  9.7
//   with the best 20     22.6 26.2  26.5 29.9     13.9 13.7  16.2 15.1     12.5 11.6  14.4 12.7  16.2 13.2
//   distillation         19.6 23.3  23.6 26.5     12.0 13.1  13.9 14.3     10.6 10.4  12.2 11.3  13.5 11.9
// Long rows gain by up to a fifth, rows of some 60 KB lose by as much where there are many of them; one bound for all is taken at
// 444 rows, where two CTAs still fit.
inline int splits_for(long long rows, int V, int elem) {
    const int step = THREADS * 16 / elem;
    int n = 1;
    while (n < MAX_SPLITS && rows * n * 2 <= 148 * 6 && V > step * n) n *= 2;
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

inline bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }
inline int elem_size(int dtype) { return dtype == LME_F32 ? 4 : 2; }
// Steps of a gradient's CTA: eight where that still makes many CTAs, so that what it has to know of its row costs little, else
// four, fewer where SMs would be idle (distillation at 8192 x 128256 bf16, backward: 644 us; sixteen steps: 674; at 2047 x
// 50257: 78, with sixteen 76).
struct GradGrid {
    int chunks, steps;
};
inline GradGrid grad_grid(long long rows, int V, int elem) {
    const int n = 16 / elem, step = THREADS * UNROLL;
    const int vectors = static_cast<int>((V + 2ll * n - 2) / n), all = (vectors + step - 1) / step;   // the first may be a part
    auto chunks = [&](int steps) { return (all + steps - 1) / steps; };
    int steps = rows * chunks(8) >= 148 * 40 ? 8 : 4;
    while (steps > 1 && rows * chunks(steps) < 148 * 8) steps /= 2;
    return {chunks(steps), steps};
}

// Dynamic shared memory of the streaming kernels; the attribute is set to the most that any call asks for.
constexpr int MAX_SMEM = RING_BYTES + MAX_MAP;
template <typename T>
inline cudaError_t launch_score(const ScoreArgs& a, long long ctas, void* stream) {
    const bool top = a.k > 0;
    const int smem = max(RING_BYTES, top ? static_cast<int>(sizeof(Selection)) : 0);
    if (!(top ? opt_in<token_logprobs_kernel<T, true>>(cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM)
              : opt_in<token_logprobs_kernel<T, false>>(cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM)))
        return cudaErrorInvalidValue;
    return top ? launch(token_logprobs_kernel<T, true>, a, ctas, a.splits, smem, stream)
               : launch(token_logprobs_kernel<T, false>, a, ctas, a.splits, smem, stream);
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
    if (V > MAX_V || rows > MAX_GRID) return LME_ERR_TOO_LARGE;
    const int splits = splits_for(rows, V, elem_size(dtype));
    if (rows * splits > MAX_GRID) return LME_ERR_TOO_LARGE;
    if (x == nullptr || entropy == nullptr || (tokens != nullptr && logprobs == nullptr) ||
        (k > 0 && (top_logprobs == nullptr || top_ids == nullptr)))
        return LME_ERR_SHAPE;
    if (misaligned(stats)) return LME_ERR_ALIGN;
    const ScoreArgs a{{x, inner, ld_inner, ld_outer, V}, tokens, ignore_index, 1.0 / temperature, k, splits, logprobs, entropy,
                      top_logprobs, top_ids, stats};
    const long long ctas = rows * splits;
    const cudaError_t e = dtype == LME_BF16  ? launch_score<__nv_bfloat16>(a, ctas, stream)
                          : dtype == LME_F16 ? launch_score<__half>(a, ctas, stream)
                                             : launch_score<float>(a, ctas, stream);
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
    if (V > MAX_V) return LME_ERR_TOO_LARGE;
    const GradGrid grid = grad_grid(rows, V, elem_size(dtype));
    if (rows * grid.chunks > MAX_GRID) return LME_ERR_TOO_LARGE;
    if (x == nullptr || grad == nullptr || stats == nullptr || (d_top != nullptr && top_ids == nullptr)) return LME_ERR_SHAPE;
    if (misaligned(stats)) return LME_ERR_ALIGN;
    const ScoreGradArgs a{{x, inner, ld_inner, ld_outer, V}, grad, tokens, ignore_index, static_cast<float>(1.0 / temperature), k,
                          grid.chunks, grid.steps, stats, top_ids, d_logprobs, d_entropy, d_top};
    const long long ctas = rows * grid.chunks;
    const cudaError_t e = dtype == LME_BF16  ? launch(token_logprobs_grad_kernel<__nv_bfloat16>, a, ctas, 1, 0, stream)
                          : dtype == LME_F16 ? launch(token_logprobs_grad_kernel<__half>, a, ctas, 1, 0, stream)
                                             : launch(token_logprobs_grad_kernel<float>, a, ctas, 1, 0, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}

namespace lme {
namespace vr {
inline AtOne at_one(bool labels, double temperature) { return !labels || temperature == 1.0 ? NONE : temperature == 2.0 ? SQUARE : OWN; }
template <typename T, AtOne ONE>
inline cudaError_t launch_distill_one(const DistillArgs& a, long long ctas, int smem, void* stream) {
    if (!opt_in<topk_distillation_kernel<T, ONE>>(cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM)) return cudaErrorInvalidValue;
    return launch(topk_distillation_kernel<T, ONE>, a, ctas, a.splits, smem, stream);
}
template <typename T>
inline cudaError_t launch_distill(const DistillArgs& a, AtOne one, long long ctas, int smem, void* stream) {
    return one == NONE  ? launch_distill_one<T, NONE>(a, ctas, smem, stream)
           : one == OWN ? launch_distill_one<T, OWN>(a, ctas, smem, stream)
                        : launch_distill_one<T, SQUARE>(a, ctas, smem, stream);
}
template <typename T>
inline cudaError_t launch_distill_grad(const DistillGradArgs& a, AtOne one, long long ctas, void* stream) {
    return one == NONE  ? launch(topk_distillation_grad_kernel<T, NONE>, a, ctas, 1, 0, stream)
           : one == OWN ? launch(topk_distillation_grad_kernel<T, OWN>, a, ctas, 1, 0, stream)
                        : launch(topk_distillation_grad_kernel<T, SQUARE>, a, ctas, 1, 0, stream);
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
    if (V > MAX_V || rows > MAX_GRID) return LME_ERR_TOO_LARGE;
    const int n = 16 / elem_size(dtype);
    int splits = splits_for(rows, V, elem_size(dtype));
    auto map_bytes = [&](int s) { return ((((V + 2 * n - 2) / n + s - 1) / s + WARP_STEP - 1) / WARP_STEP * 32 + 4) * 4; };
    while (splits < MAX_SPLITS && map_bytes(splits) > MAX_MAP) splits *= 2;
    if (map_bytes(splits) > MAX_MAP || rows * splits > MAX_GRID) return LME_ERR_TOO_LARGE;
    if (x == nullptr || top_ids == nullptr || top_logprobs == nullptr || kl == nullptr || entries == nullptr || stats == nullptr)
        return LME_ERR_SHAPE;
    if (misaligned(stats)) return LME_ERR_ALIGN;
    const DistillArgs a{{x, inner, ld_inner, ld_outer, V}, top_ids, top_logprobs, labels, ignore_index, 1.0 / temperature, k,
                        splits, forward_kl, tail, kl, nll, entries, stats};
    const AtOne one = at_one(labels != nullptr, temperature);
    const long long ctas = rows * splits;
    const int smem = RING_BYTES + map_bytes(splits);
    const cudaError_t e = dtype == LME_BF16  ? launch_distill<__nv_bfloat16>(a, one, ctas, smem, stream)
                          : dtype == LME_F16 ? launch_distill<__half>(a, one, ctas, smem, stream)
                                             : launch_distill<float>(a, one, ctas, smem, stream);
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
    if (V > MAX_V) return LME_ERR_TOO_LARGE;
    const GradGrid grid = grad_grid(rows, V, elem_size(dtype));
    if (rows * grid.chunks > MAX_GRID) return LME_ERR_TOO_LARGE;
    if (x == nullptr || grad == nullptr || stats == nullptr || entries == nullptr || top_logprobs == nullptr) return LME_ERR_SHAPE;
    if (misaligned(stats)) return LME_ERR_ALIGN;
    const DistillGradArgs a{{x, inner, ld_inner, ld_outer, V}, grad, entries, top_logprobs, labels, ignore_index,
                            static_cast<float>(1.0 / temperature), k, grid.chunks, grid.steps, forward_kl, stats, d_kl, d_nll};
    const AtOne one = at_one(d_nll != nullptr, temperature);
    const long long ctas = rows * grid.chunks;
    const cudaError_t e = dtype == LME_BF16  ? launch_distill_grad<__nv_bfloat16>(a, one, ctas, stream)
                          : dtype == LME_F16 ? launch_distill_grad<__half>(a, one, ctas, stream)
                                             : launch_distill_grad<float>(a, one, ctas, stream);
    return e == cudaSuccess ? LME_LAUNCH_OK() : LME_ERR_LAUNCH;
}
