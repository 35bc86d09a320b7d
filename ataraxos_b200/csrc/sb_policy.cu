// sb_policy.cu -- operators on rows of policy logits under a legal-action
// mask: log-probabilities of given actions with entropy and top alternatives,
// and the divergence from a teacher's listed actions, both with gradients.
//
// Mathematics, per row with legal set L and temperature T:
//   M = max_L x, d_a = (x_a - M) / T, Z = sum_L exp(d_a), log p_a = d_a - log Z
//   entropy H = log Z - (sum_L exp(d_a) d_a) / Z
// One pass keeps (M, n, r, t): n entries equal to M, r = sum of exp(d) over
// the others, t = sum of exp(d) d.  Holding the maximum's own 1 apart from r
// keeps log Z = log1p((n - 1) + r) exact to its last bits when one action
// holds nearly all of the mass.  Sums are float32; exponentials are base 2
// with log2(e) / T folded into the factor of x - M (the difference is taken
// first, so large logits lose nothing).
//
// Layout of the work: a row belongs to one warp, or to the four warps of a
// CTA where it is long (wide_forward, wide_backward).  That rule looks at the
// shape and the types alone, so a row's bits do not depend on the batch it
// comes in.  A legal mask is
// staged in shared memory as one bit per action, and only the logits of set
// bits are read: a position has some 30 legal moves of 10,000, so a row costs
// its mask and 30 sectors instead of 20 or 40 KB.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "sb_error.h"
#include "stratego_b200.h"

namespace sb {
namespace {

constexpr int WARPS = 4;                  // warps of a CTA: one row each, or one row together
constexpr unsigned ALL = 0xffffffffu;
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int LIST = 1024;                // legal actions a warp gathers at once
constexpr int BLOCK_WORDS = 11;           // mask words of a lane between two gathers (odd: no bank conflicts)
constexpr int CHUNKS = 64;                // gradient chunks a warp lists at once
constexpr int SLOT = 48;                  // bytes between two lanes' chunk slots (32 used)

struct Rows {
    const void* x;
    const uint8_t* mask;
    int64_t n, stride, mask_stride;
    int a;
    float inv_t;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float exp2_(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}

// A chunk is 32 bytes of a row (one DRAM sector): 16 or 8 elements.
template <typename T> struct Chunk {
    static constexpr int E = 32 / sizeof(T);
    uint32_t w[8];
    __device__ __forceinline__ void load(const T* p) {
        asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(p));
    }
    __device__ __forceinline__ void store(T* p) const {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                     "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    }
    __device__ __forceinline__ void fill(uint32_t v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = v;
    }
    __device__ __forceinline__ float get(int e) const;
    __device__ __forceinline__ void set(int e, float v);
};
template <> __device__ __forceinline__ float Chunk<float>::get(int e) const { return __uint_as_float(w[e]); }
template <> __device__ __forceinline__ void Chunk<float>::set(int e, float v) { w[e] = __float_as_uint(v); }
template <> __device__ __forceinline__ float Chunk<__nv_bfloat16>::get(int e) const {
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
}
template <> __device__ __forceinline__ void Chunk<__nv_bfloat16>::set(int e, float v) {
    const uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | b << 16 : (w[e >> 1] & 0xffff0000u) | b;
}
template <> __device__ __forceinline__ float Chunk<__half>::get(int e) const {
    return __half2float(__ushort_as_half((unsigned short)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu)));
}
template <> __device__ __forceinline__ void Chunk<__half>::set(int e, float v) {
    const uint32_t b = __half_as_ushort(__float2half_rn(v));
    w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | b << 16 : (w[e >> 1] & 0xffff0000u) | b;
}

__device__ __forceinline__ int64_t load_index(const void* p, int bytes, int64_t i) {
    if (bytes == 8) return static_cast<const int64_t*>(p)[i];
    if (bytes == 4) return static_cast<const int32_t*>(p)[i];
    return static_cast<const int16_t*>(p)[i];
}

__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t i) {
    if (dtype == SB_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == SB_DTYPE_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_f(static_cast<const __half*>(p)[i]);
}

// ---- legal bits in shared memory -------------------------------------------

// Bit a + P of `w` is 1 where action a is legal; words before and after the
// row are 0, so a field that reaches past either end reads zeros.
struct Bits {
    uint32_t* w;
    int p;
    __device__ __forceinline__ bool test(int a) const { return (w[(a + p) >> 5] >> ((a + p) & 31)) & 1; }
    // the 32 actions from 32 i on
    __device__ __forceinline__ uint32_t word(int i) const {
        const int b = 32 * i + p;
        return __funnelshift_r(w[b >> 5], w[(b >> 5) + 1], b & 31);
    }
    // `len` <= 16 bits of the actions from a on (a >= -16)
    __device__ __forceinline__ uint32_t field(int a, int len) const {
        const int b = a + p;
        return __funnelshift_r(w[b >> 5], w[(b >> 5) + 1], b & 31) & ((1u << len) - 1u);
    }
};

// Bytes of a staged row: the bits, 32 of lead (16 to align a bit-packed row's
// chunks, 16 of zeros) and zeros past the end.
__host__ __device__ constexpr int bits_bytes(int a) { return ((a + 7) / 8 + 32 + 48 + 15) / 16 * 16; }

__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t v) {  // bit i: byte i of v is not 0
    const uint32_t t = (((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) & 0x80808080u;
    return ((t >> 7) * 0x01020408u) >> 24 & 15u;
}

// Stage one row's mask with G threads (tid 0..G-1; the caller synchronises).
template <int MASK, int G>
__device__ __forceinline__ Bits stage(uint8_t* sh, const uint8_t* m, int a, int tid) {
    const int h = (int)(-(intptr_t)m & 15), off = (16 - h) & 15;
    if (MASK == SB_MASK_BITS) {
        // Row byte i goes to sh[16 + off + i], so that the 16-byte chunks of
        // the row in memory stay 16-byte chunks here.  The row's last byte is
        // always handled as a tail byte: its bits past the last action drop.
        const int len = (a + 7) >> 3, nb = len - h > 0 ? (len - h - 1) >> 4 : 0;
        uint4* s4 = reinterpret_cast<uint4*>(sh + 16 + off + h);
        const uint4* g4 = reinterpret_cast<const uint4*>(m + h);
#pragma unroll 3
        for (int j = tid; j < nb; j += G) s4[j] = __ldg(g4 + j);
        const uint8_t last = (uint8_t)(0xffu >> (-a & 7));
        for (int q = tid; q < 64; q += G) {  // 32 lead bytes (head included), then 32 tail bytes
            const int i = q < 32 ? q - 16 - off : h + 16 * nb + q - 32;
            if (q < 32 && i >= h) continue;
            uint8_t v = 0;
            if (i >= 0 && i < len) v = i == len - 1 ? m[i] & last : m[i];
            sh[16 + off + i] = v;
        }
        return {reinterpret_cast<uint32_t*>(sh), 8 * (16 + off)};
    }
    // One byte per action: 16 of them make one halfword.
    uint16_t* s2 = reinterpret_cast<uint16_t*>(sh);
    const int lead = 2 + (h > 0), nb = a > h ? (a - h) >> 4 : 0;
    const uint4* g4 = reinterpret_cast<const uint4*>(m + h);
#pragma unroll 5
    for (int j = tid; j < nb; j += G) {
        const uint4 v = __ldg(g4 + j);
        uint32_t b = 0;
        if (v.x | v.y | v.z | v.w)
            b = nonzero_bytes(v.x) | nonzero_bytes(v.y) << 4 | nonzero_bytes(v.z) << 8 | nonzero_bytes(v.w) << 12;
        s2[lead + j] = (uint16_t)b;
    }
    if (tid < 32) {
        const int i = tid < 16 ? tid - off : h + 16 * nb + tid - 16;
        const bool on = tid < 16 ? (i >= 0 && i < h && i < a) : i < a;
        const uint32_t b = __ballot_sync(ALL, on && m[on ? i : 0] != 0);
        if (tid < 2) s2[tid] = 0;
        if (tid == 2 && h > 0) s2[2] = (uint16_t)(b & 0xffffu);
        if (tid >= 8 && tid < 16) s2[lead + nb + tid - 8] = tid == 8 ? (uint16_t)(b >> 16) : 0;
    }
    return {reinterpret_cast<uint32_t*>(sh), 32 + off};
}

// ---- running sums ------------------------------------------------------------

// M is the same in all lanes of a warp; n, r and t are the lane's own shares.
// t is in units of log2(e): sum of exp(d) d log2(e).
struct Sum {
    float m, n, r, t;
};

// Take up a tile of N logits per lane (-inf where there is none).  A NaN
// reaches r; +inf stays the maximum; both make the row NaN at the end.
template <int N, bool ENT>
__device__ __forceinline__ void take(Sum& s, const float (&x)[N], float c) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    m = warp_max(fmaxf(m, NEG_INF));
    if (m > s.m) {
        const float d = (s.m - m) * c, f = exp2_(d), w = s.r + s.n;
        if (ENT) s.t = f * (s.t + w * fmaxf(d, -1e4f));
        s.r = f * w;
        s.n = 0.f;
        s.m = m;
    }
    const float ref = s.m == NEG_INF ? 0.f : s.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = (x[i] - ref) * c, e = exp2_(d);
        if (x[i] == ref) s.n += 1.f;
        else s.r += e;
        if (ENT) s.t = fmaf(e, fmaxf(d, -1e4f), s.t);
    }
}

__device__ __forceinline__ Sum no_sum() { return {NEG_INF, 0.f, 0.f, 0.f}; }

// Two sums as one; both in full (all lanes' shares joined).
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
    if (b.m > a.m) {
        const Sum q = a;
        a = b;
        b = q;
    }
    const bool eq = a.m == b.m;
    const float d = eq ? 0.f : (b.m - a.m) * c, f = exp2_(d), w = b.r + b.n;
    a.t += f * (b.t + (eq ? 0.f : w * fmaxf(d, -1e4f)));
    a.r += eq ? b.r : f * w;
    a.n += eq ? b.n : 0.f;
    return a;
}

// The sum of a whole row in every thread: over the warp's lanes, then over
// the row's warps by way of shared memory.
template <int W>
__device__ __forceinline__ Sum whole(Sum s, float c, Sum* sh) {
    s.n = warp_sum(s.n);
    s.r = warp_sum(s.r);
    s.t = warp_sum(s.t);
    if (W > 1) {
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
        __syncthreads();
        s = sh[0];
#pragma unroll
        for (int w = 1; w < W; ++w) s = join(s, sh[w], c);
    }
    return s;
}

// (M, log Z) as the outputs and the backward pass use them: log Z = inf for a
// row without an action of non-zero probability (every p is then 0) and NaN
// for a row that holds a legal NaN or +inf.
__device__ __forceinline__ float2 stats_of(Sum s) {
    if (s.r != s.r || s.m == INFINITY) return make_float2(0.f, NAN);
    if (s.m == NEG_INF) return make_float2(0.f, INFINITY);
    return make_float2(s.m, log1pf((s.n - 1.f) + s.r));
}

// ---- the likeliest actions ------------------------------------------------------

// A warp's best `k` entries in descending order, one per lane; ties go to the
// lower action.
struct Top {
    float x, bar_x;  // this lane's entry; the k-th one
    int a, bar_a, k;
    __device__ __forceinline__ void init(int n) {
        x = bar_x = NEG_INF;
        a = bar_a = 0x7fffffff;
        k = n;
    }
    __device__ __forceinline__ void set_bar() {
        bar_x = __shfl_sync(ALL, x, k - 1);
        bar_a = __shfl_sync(ALL, a, k - 1);
    }
    __device__ __forceinline__ bool wants(float v, int b) const {
        return v > bar_x || (v == bar_x && b < bar_a && v > NEG_INF);
    }
    // One candidate per lane (-inf: none), put in place one by one.
    __device__ __forceinline__ void offer(float v, int b) {
        unsigned c = __ballot_sync(ALL, wants(v, b));
        while (c) {
            const int src = __ffs(c) - 1;
            const float cx = __shfl_sync(ALL, v, src);
            const int ca = __shfl_sync(ALL, b, src);
            const int at = __popc(__ballot_sync(ALL, x > cx || (x == cx && a < ca)));
            const float ux = __shfl_up_sync(ALL, x, 1);
            const int ua = __shfl_up_sync(ALL, a, 1);
            const int lane = threadIdx.x & 31;
            if (lane >= at) {
                x = lane == at ? cx : ux;
                a = lane == at ? ca : ua;
            }
            set_bar();
            c &= c - 1;
            c &= __ballot_sync(ALL, wants(v, b));
        }
    }
    // The first 32 candidates of an empty list: a bitonic sort (15 exchanges
    // instead of up to 32 insertions).
    __device__ __forceinline__ void fill(float v, int b) {
        const int lane = threadIdx.x & 31;
        x = v == v ? v : NEG_INF;
        a = x > NEG_INF ? b : 0x7fffffff;
#pragma unroll
        for (int n = 2; n <= 32; n <<= 1) {
#pragma unroll
            for (int d = n >> 1; d; d >>= 1) {
                const float ox = __shfl_xor_sync(ALL, x, d);
                const int oa = __shfl_xor_sync(ALL, a, d);
                const bool mine_first = x > ox || (x == ox && a < oa);
                const bool keep_first = ((lane & d) == 0) == ((lane & n) == 0);
                if (mine_first != keep_first) {
                    x = ox;
                    a = oa;
                }
            }
        }
        set_bar();
    }
};

// ---- one pass over a row ------------------------------------------------------------

// The legal logits of this warp's blocks of a row (block b is warp b % W's).
// The legal actions are listed in ascending order and dealt to the lanes in
// turn, so the sums' order, and with it every bit of the result, is the same
// for any kind of mask and wherever its rows lie.  SKIP leaves out the
// actions of `skip`.  Returns how many actions were taken.
template <typename T, int W, bool ENT, bool TOP, bool SKIP>
__device__ __forceinline__ int pass_masked(Sum& s, Top& top, const T* x, Bits bits, Bits skip, int a, float c,
                                           uint16_t* list, int part) {
    const int lane = threadIdx.x & 31;
    const int words = (a + 31) >> 5;
    auto word = [&](int i) { return i >= words ? 0u : SKIP ? bits.word(i) & ~skip.word(i) : bits.word(i); };
    int taken = 0;
    for (int w0 = part * 32 * BLOCK_WORDS; w0 < words; w0 += 32 * BLOCK_WORDS * W) {
        const int mine = w0 + lane * BLOCK_WORDS;
        uint32_t some = 0;  // bit k: the lane's word k is not 0
        int count = 0;
#pragma unroll
        for (int k = 0; k < BLOCK_WORDS; ++k) {
            const uint32_t w = word(mine + k);
            count += __popc(w);
            some |= w ? 1u << k : 0u;
        }
        int at = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(ALL, at, o);
            if (lane >= o) at += v;
        }
        const int total = __shfl_sync(ALL, at, 31);
        if (total == 0) continue;
        const bool first = taken == 0;
        taken += total;
        if (total <= LIST) {
            at -= count;
            uint32_t w = 0;
            int base = 0;
            while (some | w) {  // one action a turn, whichever word it is in
                if (!w) {
                    const int i = mine + __ffs(some) - 1;
                    some &= some - 1;
                    w = word(i);
                    base = i * 32;
                }
                list[at++] = (uint16_t)(base + __ffs(w) - 1);
                w &= w - 1;
            }
            __syncwarp();
            if (TOP || total <= 32) {
                for (int i = 0; i < total; i += 32) {
                    const int b = i + lane < total ? list[i + lane] : 0;
                    const float v[1] = {i + lane < total ? to_f(x[b]) : NEG_INF};
                    take<1, ENT>(s, v, c);
                    if (TOP) {
                        if (first && i == 0) top.fill(v[0], b);
                        else top.offer(v[0], b);
                    }
                }
            } else {
                for (int i = 0; i < total; i += 128) {
                    float v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int n = i + q * 32 + lane;
                        v[q] = n < total ? to_f(x[list[n]]) : NEG_INF;
                    }
                    take<4, ENT>(s, v, c);
                }
            }
            __syncwarp();
        } else {
            // too many for the list: every word's 32 actions in turn, a lane each
            const int end = min(words, w0 + 32 * BLOCK_WORDS);
            float best = NEG_INF;
            for (int i = w0; i < end; i += 8) {
                float v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint32_t m = i + q < end ? word(i + q) : 0u;
                    v[q] = (m >> lane) & 1 ? to_f(x[(i + q) * 32 + lane]) : NEG_INF;
                    best = fmaxf(best, v[q]);
                }
                take<8, ENT>(s, v, c);
            }
            if (TOP) {
                // only a lane whose best reaches the k-th best of what the list
                // holds and of all lanes' bests can hold one of the k best
                Top bar = top;
                bar.offer(best, lane);
                unsigned who = __ballot_sync(ALL, best >= bar.bar_x && best > NEG_INF);
                for (; who; who &= who - 1) {
                    const int src = __ffs(who) - 1;
                    for (int i = w0; i < end; i += 32) {
                        const int b = (i + lane) * 32 + src;
                        const uint32_t m = i + lane < end ? word(i + lane) : 0u;
                        top.offer((m >> src) & 1 ? to_f(x[b]) : NEG_INF, b);
                    }
                }
            }
        }
    }
    return taken;
}

// The same without a mask: 32-byte chunks of the row at their alignment in
// memory, the ends that do not fill one by single loads.  Returns the lane's
// largest logit.
template <typename T> struct Span {
    int head, chunks;
    __device__ __forceinline__ Span(const T* x, int a) {
        head = min(a, (int)((-(intptr_t)x & 31) / sizeof(T)));
        chunks = (a - head) / Chunk<T>::E;
    }
};

template <typename T, int W, bool ENT, bool SKIP>
__device__ __forceinline__ float pass_all(Sum& s, const T* x, Bits skip, int a, float c, int part) {
    constexpr int E = Chunk<T>::E, U = 32 / E;
    const int lane = threadIdx.x & 31;
    const Span<T> sp(x, a);
    float best = NEG_INF;
    if (part == 0) {  // the ends: fewer than two chunks, one element a lane
        const int b = lane < sp.head ? lane : sp.chunks * E + lane;
        const float v[1] = {b < a && !(SKIP && skip.test(b)) ? to_f(x[b]) : NEG_INF};
        best = fmaxf(best, v[0]);
        take<1, ENT>(s, v, c);
    }
    const T* body = x + sp.head;
    for (int c0 = part * 32; c0 < sp.chunks; c0 += 32 * U * W) {
        float v[32];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = c0 + u * 32 * W + lane;
            Chunk<T> q;
            if (i < sp.chunks) {
                q.load(body + i * E);
                const uint32_t out = SKIP ? skip.field(sp.head + i * E, E) : 0u;
#pragma unroll
                for (int e = 0; e < E; ++e) v[u * E + e] = SKIP && (out >> e) & 1 ? NEG_INF : q.get(e);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[u * E + e] = NEG_INF;
            }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) best = fmaxf(best, v[i]);
        take<32, ENT>(s, v, c);
    }
    return best;
}

// The k best of an unmasked row, by one warp: `best[W * 32]` holds every
// lane's largest logit.  The k-th largest of those bounds the k-th best of the
// row from below, so only the lanes that reach it are looked through again
// (about k of them, from cache).
template <typename T, int W>
__device__ __forceinline__ void top_of_all(Top& top, const T* x, int a, const float* best) {
    constexpr int E = Chunk<T>::E;
    const int lane = threadIdx.x & 31;
    const Span<T> sp(x, a);
    Top bar = top;
    bar.fill(best[lane], lane);
#pragma unroll
    for (int w = 1; w < W; ++w) bar.offer(best[w * 32 + lane], w * 32 + lane);
    for (int w = 0; w < W; ++w) {
        const float mine = best[w * 32 + lane];
        unsigned who = __ballot_sync(ALL, mine >= bar.bar_x && mine > NEG_INF);
        for (; who; who &= who - 1) {
            const int src = __ffs(who) - 1;
            // its chunks are w * 32 + src + n * 32 * W, E elements of each
            for (int i = lane; __any_sync(ALL, w * 32 + src + i / E * 32 * W < sp.chunks); i += 32) {
                const int ch = w * 32 + src + i / E * 32 * W, b = sp.head + ch * E + i % E;
                const float v = ch < sp.chunks ? to_f(x[b]) : NEG_INF;
                top.offer(v >= bar.bar_x ? v : NEG_INF, b);
            }
            if (w == 0) {  // and its element of the row's ends
                const int b = src < sp.head ? src : sp.chunks * E + src;
                top.offer(lane == 0 && b < a ? to_f(x[b]) : NEG_INF, b);
            }
        }
    }
}

// ---- forward: given actions, entropy, top alternatives -----------------------------

template <typename T, int MASK, int W, bool TOP>
__global__ void __launch_bounds__(WARPS * 32) logprobs_kernel(Rows R, sb_logprobs o) {
    extern __shared__ uint4 dyn[];
    __shared__ Sum sums[WARPS];
    __shared__ float top_x[WARPS][32];
    __shared__ int top_a[WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* sh = reinterpret_cast<uint8_t*>(dyn);
    const int row_bytes = MASK == SB_MASK_NONE ? 0 : bits_bytes(R.a);
    uint8_t* sh_bits = sh + (W == 1 ? warp * row_bytes : 0);
    uint16_t* list = reinterpret_cast<uint16_t*>(sh + (WARPS / W) * row_bytes) + warp * LIST;
    const float c = R.inv_t * LOG2E;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        int64_t act = -1;
        float xa = 0.f;
        if (o.actions) {
            act = load_index(o.actions, o.action_bytes, row);
            if (act >= 0 && act < R.a) xa = to_f(x[act]);
        }
        Sum s = no_sum();
        Top top;
        top.init(TOP ? o.top : 1);
        bool legal = act >= 0 && act < R.a;
        if (MASK == SB_MASK_NONE) {
            const float best = pass_all<T, W, true, false>(s, x, Bits{}, R.a, c, W == 1 ? 0 : warp);
            if (TOP) {
                top_x[warp][lane] = best;
                if (W == 1) __syncwarp();
            }
        } else {
            const Bits bits = stage<MASK, 32 * W>(sh_bits, R.mask + row * R.mask_stride, R.a, W == 1 ? lane : threadIdx.x);
            if (W == 1) __syncwarp();
            else __syncthreads();
            legal = legal && bits.test((int)act);
            pass_masked<T, W, true, TOP, false>(s, top, x, bits, bits, R.a, c, list, W == 1 ? 0 : warp);
        }
        if (TOP && W > 1 && MASK != SB_MASK_NONE) {
            top_x[warp][lane] = top.x;
            top_a[warp][lane] = top.a;
        }
        s = whole<W>(s, c, sums);
        const float2 st = stats_of(s);
        if (W == 1 || warp == 0) {
            if (lane == 0) {
                if (o.logprob) o.logprob[row] = act == -1 ? 0.f : legal ? (xa - st.x) * R.inv_t - st.y : NEG_INF;
                o.entropy[row] = st.y == INFINITY ? 0.f : st.y - LN2 * s.t / (s.n + s.r);
                if (o.row_stats) *reinterpret_cast<float2*>(o.row_stats + 2 * row) = st;
            }
            if (TOP) {
                if (MASK == SB_MASK_NONE)
                    top_of_all<T, W>(top, x, R.a, top_x[W == 1 ? warp : 0]);
                else if (W > 1)
                    for (int w = 1; w < W; ++w) top.offer(lane < o.top ? top_x[w][lane] : NEG_INF, top_a[w][lane]);
                if (lane < o.top) {
                    const bool some = top.x > NEG_INF;
                    o.top_action[row * o.top + lane] = some ? top.a : -1;
                    o.top_logprob[row * o.top + lane] =
                        st.y != st.y ? NAN : some ? (top.x - st.x) * R.inv_t - st.y : NEG_INF;
                }
            }
        }
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

// ---- gradient rows ---------------------------------------------------------------------

// Gradient of a row: p (c0 + c1 log p) / T off the listed actions, and
// (p (l0 + c1 log p) + the sum of its entries' shares) / T on them.
struct RowGrad {
    float m, logz, c0, c1, l0;
};

template <bool ENT>
__device__ __forceinline__ float grad_of(float x, const RowGrad& g, float c0, float add, float inv_t) {
    const float lp = (x - g.m) * inv_t - g.logz, p = exp2_(lp * LOG2E);
    // p is 0 below -104: the bound keeps 0 * inf out and changes nothing else
    return (p * (ENT ? c0 + g.c1 * fmaxf(lp, -1e4f) : c0) + add) * inv_t;
}

// One lane's chunk of a gradient row: the elements that are set in `field`,
// the others 0.  Few are set: a loop over them, with the lane's slots in
// shared memory to index by.
template <typename T, bool ENT>
__device__ __forceinline__ void grad_sparse(const T* x, T* g, int first, int a, uint32_t field, const RowGrad& r,
                                            float inv_t, T* xs, T* gs) {
    constexpr int E = Chunk<T>::E;
    const bool full = first >= 0 && first + E <= a, wide = full && ((intptr_t)(x + first) & 31) == 0;
    uint4* x4 = reinterpret_cast<uint4*>(xs);
    uint4* g4 = reinterpret_cast<uint4*>(gs);
    Chunk<T> q;
    if (wide) {
        q.load(x + first);
        x4[0] = make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]);
        x4[1] = make_uint4(q.w[4], q.w[5], q.w[6], q.w[7]);
    }
    g4[0] = g4[1] = make_uint4(0, 0, 0, 0);
    asm volatile("" ::: "memory");  // the slots are read by another type than they are written by
    for (uint32_t f = field; f; f &= f - 1) {
        const int e = __ffs(f) - 1;
        gs[e] = from_f<T>(grad_of<ENT>(to_f(wide ? xs[e] : x[first + e]), r, r.c0, 0.f, inv_t));
    }
    asm volatile("" ::: "memory");
    if (full) {
        const uint4 u = g4[0], v = g4[1];
        q.w[0] = u.x, q.w[1] = u.y, q.w[2] = u.z, q.w[3] = u.w;
        q.w[4] = v.x, q.w[5] = v.y, q.w[6] = v.z, q.w[7] = v.w;
        q.store(g + first);
    } else {
        for (int e = max(0, -first); e < E && first + e < a; ++e) g[first + e] = gs[e];
    }
}

// The same with every action legal.
template <typename T, bool ENT>
__device__ __forceinline__ void grad_dense(const T* x, T* g, int first, int a, const RowGrad& r, float inv_t) {
    constexpr int E = Chunk<T>::E;
    Chunk<T> q;
    if (first >= 0 && first + E <= a) {
        if (((intptr_t)(x + first) & 31) == 0) {
            q.load(x + first);
        } else {
            q.fill(0);
#pragma unroll
            for (int e = 0; e < E; ++e) q.set(e, to_f(x[first + e]));
        }
#pragma unroll
        for (int e = 0; e < E; ++e) q.set(e, grad_of<ENT>(q.get(e), r, r.c0, 0.f, inv_t));
        q.store(g + first);
    } else {
        for (int b = max(0, first); b < first + E && b < a; ++b)
            g[b] = from_f<T>(grad_of<ENT>(to_f(x[b]), r, r.c0, 0.f, inv_t));
    }
}

// Shared memory of a warp's gradient work: the list and two slots a lane.
constexpr int GRAD_BYTES = 4 * CHUNKS + 2 * 32 * SLOT;

// A warp's part of a gradient row: the 32-byte chunks of the row as it lies
// in memory, so that every sector but the row's first and last is stored
// whole and once.  Chunks without a legal action are zeros; the others are
// listed and computed 32 at a time.  Returns the part's actions [lo, hi).
template <typename T, int MASK, int W, bool ENT>
__device__ __forceinline__ int2 grad_row(const T* x, T* g, Bits bits, int a, const RowGrad& r, float inv_t,
                                         uint8_t* sh, int part) {
    constexpr int E = Chunk<T>::E;
    const int lane = threadIdx.x & 31;
    const int e0 = (int)(((intptr_t)g & 31) / sizeof(T));
    const int chunks = (a + e0 + E - 1) / E, per = (chunks + W - 1) / W;
    const int lo = part * per, hi = min(chunks, lo + per);
    if (MASK == SB_MASK_NONE) {
        for (int ch = lo + lane; ch < hi; ch += 32) grad_dense<T, ENT>(x, g, ch * E - e0, a, r, inv_t);
    } else {
        uint32_t* list = reinterpret_cast<uint32_t*>(sh);
        T* xs = reinterpret_cast<T*>(sh + 4 * CHUNKS + lane * SLOT);
        T* gs = reinterpret_cast<T*>(sh + 4 * CHUNKS + (32 + lane) * SLOT);
        Chunk<T> zero;
        zero.fill(0);
        int count = 0;
        for (int c0 = lo; c0 < hi; c0 += 32) {
            const int ch = c0 + lane, first = ch * E - e0;
            const uint32_t f = ch < hi ? bits.field(first, E) : 0u;
            const bool full = first >= 0 && first + E <= a;
            const bool put = ch < hi && (f != 0 || !full);
            const unsigned b = __ballot_sync(ALL, put);
            if (put) list[count + __popc(b & ((1u << lane) - 1u))] = (uint32_t)ch | f << 16;
            else if (ch < hi) zero.store(g + first);
            count += __popc(b);
            if (count > CHUNKS - 32 || c0 + 32 >= hi) {
                __syncwarp();
                for (int i = lane; i < count; i += 32) {
                    const uint32_t v = list[i];
                    grad_sparse<T, ENT>(x, g, (int)(v & 0xffffu) * E - e0, a, v >> 16, r, inv_t, xs, gs);
                }
                __syncwarp();
                count = 0;
            }
        }
    }
    __syncwarp();  // the listed actions' own values are stored over these
    return make_int2(max(0, lo * E - e0), hi * E - e0);
}

template <typename T, int MASK, int W>
__global__ void __launch_bounds__(WARPS * 32) logprobs_backward_kernel(Rows R, sb_logprobs f, sb_logprobs_grad g) {
    extern __shared__ uint4 dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* sh = reinterpret_cast<uint8_t*>(dyn);
    const int row_bytes = MASK == SB_MASK_NONE ? 0 : bits_bytes(R.a);
    uint8_t* sh_bits = sh + (W == 1 ? warp * row_bytes : 0);
    uint8_t* work = sh + (WARPS / W) * row_bytes + warp * GRAD_BYTES;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        T* out = static_cast<T*>(g.grad) + row * R.a;
        // lane k < top holds alternative k; the given action's share joins the
        // alternative that is the same action, or stays alone
        int mine = -1;
        float add = 0.f;
        if (g.g_top && lane < f.top) {
            mine = (int)f.top_action[row * f.top + lane];
            if (mine >= 0) add = g.g_top[row * f.top + lane];
        }
        int64_t act = -1;
        float ga = 0.f;
        if (g.g_logprob) {
            act = load_index(f.actions, f.action_bytes, row);
            ga = g.g_logprob[row * g.g_logprob_stride];
        }
        const float gh = g.g_entropy ? g.g_entropy[row * g.g_entropy_stride] : 0.f;
        const float2 st = *reinterpret_cast<const float2*>(f.row_stats + 2 * row);
        const float h = f.entropy[row];
        Bits bits = {nullptr, 0};
        if (MASK != SB_MASK_NONE) {
            bits = stage<MASK, 32 * W>(sh_bits, R.mask + row * R.mask_stride, R.a, W == 1 ? lane : threadIdx.x);
            if (W == 1) __syncwarp();
            else __syncthreads();
        }
        bool legal = act >= 0 && act < R.a;
        if (MASK != SB_MASK_NONE) legal = legal && bits.test((int)act);
        const float total = warp_sum(add) + (legal ? ga : 0.f);
        const RowGrad r = {st.x, st.y, -(total + gh * h), -gh, -(total + gh * h)};
        const int2 own = grad_row<T, MASK, W, true>(x, out, bits, R.a, r, R.inv_t, work, W == 1 ? 0 : warp);
        const bool same = legal && mine == (int)act;
        if (same) add += ga;
        if (mine >= own.x && mine < own.y) out[mine] = from_f<T>(grad_of<true>(to_f(x[mine]), r, r.l0, add, R.inv_t));
        if (!__any_sync(ALL, same) && lane == 0 && legal && act >= own.x && act < own.y)
            out[act] = from_f<T>(grad_of<true>(to_f(x[act]), r, r.l0, ga, R.inv_t));
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

// ---- distillation ------------------------------------------------------------------------

// Kept per row for the backward pass: (M, log Z), (Q, Q - q_r / p_r) and the
// teacher's own (maximum, log sum).

// Teacher entry k of a row: its action (-1 where it is left out) and logit.
template <int MASK>
__device__ __forceinline__ int teacher(const Rows& R, const sb_distill& d, Bits bits, int64_t row, int k, float* v) {
    if (k >= d.listed) return -1;
    const int64_t a = load_index(d.teacher_actions, d.action_bytes, row * d.listed + k);
    *v = load_value(d.teacher_logits, d.teacher_dtype, row * d.listed + k);
    if (a < 0 || a >= R.a || *v == NEG_INF) return -1;
    if (MASK != SB_MASK_NONE && !bits.test((int)a)) return -1;
    return (int)a;
}

// Loss: one pass for the row's (M, Z), then the teacher's entries by one warp.
// With the tail, the unlisted actions' own mass p_r is 1 - sum p while that
// keeps its digits (sum p < 1/2), nothing where every legal action is listed,
// and otherwise summed by a second pass that leaves the listed ones out.
template <typename T, int MASK, int W, bool TAIL>
__global__ void __launch_bounds__(WARPS * 32) distill_kernel(Rows R, sb_distill d) {
    extern __shared__ uint4 dyn[];
    __shared__ Sum sums[WARPS];
    __shared__ int counts[WARPS];
    __shared__ int again;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = W == 1 ? lane : threadIdx.x;
    const int part = W == 1 ? 0 : warp;
    uint8_t* sh = reinterpret_cast<uint8_t*>(dyn);
    const int row_bytes = bits_bytes(R.a) * ((MASK != SB_MASK_NONE) + TAIL);
    uint8_t* sh_bits = sh + (W == 1 ? warp * row_bytes : 0);
    uint32_t* sh_skip = reinterpret_cast<uint32_t*>(sh_bits + (MASK != SB_MASK_NONE ? bits_bytes(R.a) : 0));
    uint16_t* list = reinterpret_cast<uint16_t*>(sh + (WARPS / W) * row_bytes) + warp * LIST;
    const float c = R.inv_t * LOG2E, tc = TAIL ? 1.f : R.inv_t;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        Bits bits = {nullptr, 0};
        if (MASK != SB_MASK_NONE) bits = stage<MASK, 32 * W>(sh_bits, R.mask + row * R.mask_stride, R.a, tid);
        if (TAIL)
            for (int i = tid; i < bits_bytes(R.a) / 4; i += 32 * W) sh_skip[i] = 0;
        if (W == 1) __syncwarp();
        else __syncthreads();
        const Bits skip = {sh_skip, bits.p};
        Sum s = no_sum();
        Top none;
        int legal = 0;
        if (MASK == SB_MASK_NONE) pass_all<T, W, false, false>(s, x, skip, R.a, c, part);
        else legal = pass_masked<T, W, false, false, false>(s, none, x, bits, bits, R.a, c, list, part);
        if (W > 1 && lane == 0) counts[warp] = legal;
        s = whole<W>(s, c, sums);
        if (W > 1) {
            legal = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) legal += counts[w];
        }
        if (MASK == SB_MASK_NONE) legal = R.a;
        const float2 st = stats_of(s);
        float loss = 0.f, total = 0.f, share = 0.f;
        float2 tst = make_float2(0.f, 0.f);
        bool more = false;  // a second pass is needed
        if (W == 1 || warp == 0) {
            if (!TAIL) {
                Sum ts = no_sum();
                for (int k0 = 0; k0 < d.listed; k0 += 32) {
                    float v = 0.f;
                    const int a = teacher<MASK>(R, d, bits, row, k0 + lane, &v);
                    const float t[1] = {a >= 0 ? v : NEG_INF};
                    take<1, false>(ts, t, c);
                }
                tst = stats_of(whole<1>(ts, c, nullptr));
            }
            float sp = 0.f;
            int unique = 0;
            for (int k0 = 0; k0 < d.listed; k0 += 32) {
                float v = 0.f, p = 0.f;
                const int a = teacher<MASK>(R, d, bits, row, k0 + lane, &v);
                if (a >= 0) {
                    const float lq = (v - tst.x) * tc - tst.y, q = expf(lq), lp = (to_f(x[a]) - st.x) * R.inv_t - st.y;
                    loss += q > 0.f || q != q ? q * (lq - lp) : 0.f;
                    total += q;
                    p = expf(lp);
                }
                if (TAIL) {  // an action's first entry stands for it in p
                    const unsigned peers = __match_any_sync(ALL, a);
                    const bool lead = a >= 0 && (peers & ((1u << lane) - 1u)) == 0 && !skip.test(a);
                    __syncwarp();
                    if (lead) {
                        sp += p;
                        atomicOr(&sh_skip[(a + skip.p) >> 5], 1u << ((a + skip.p) & 31));
                    }
                    unique += __popc(__ballot_sync(ALL, lead));
                    __syncwarp();
                }
            }
            loss = warp_sum(loss);
            total = warp_sum(total);
            if (TAIL) {
                sp = warp_sum(sp);
                const float qr = legal > unique ? fmaxf(0.f, 1.f - total) : 0.f;
                more = qr > 0.f && !(sp < 0.5f);
                if (qr > 0.f && !more) {
                    const float lqr = log1pf(-total), lpr = log1pf(-sp);
                    loss += qr * (lqr - lpr);
                    share = expf(lqr - lpr);
                    total += qr;
                }
            }
        }
        if (TAIL) {
            if (W > 1) {
                if (threadIdx.x == 0) again = more;
                __syncthreads();
                more = again;
            }
            if (more) {
                Sum rest = no_sum();
                if (MASK == SB_MASK_NONE) pass_all<T, W, false, true>(rest, x, skip, R.a, c, part);
                else pass_masked<T, W, false, false, true>(rest, none, x, bits, skip, R.a, c, list, part);
                rest = whole<W>(rest, c, sums);
                if ((W == 1 || warp == 0) && rest.m > NEG_INF) {
                    const float2 sr = stats_of(rest);
                    const float qr = fmaxf(0.f, 1.f - total), lqr = log1pf(-total);
                    const float lpr = (sr.x - st.x) * R.inv_t + sr.y - st.y;
                    loss += qr * (lqr - lpr);
                    share = expf(lqr - lpr);
                    total += qr;
                }
            }
        }
        if ((W == 1 || warp == 0) && lane == 0) {
            d.loss[row] = loss;
            if (d.row_stats) {
                float2* o = reinterpret_cast<float2*>(d.row_stats + 6 * row);
                o[0] = st;
                o[1] = make_float2(total, total - share);
                o[2] = tst;
            }
        }
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

template <typename T, int MASK, int W>
__global__ void __launch_bounds__(WARPS * 32) distill_backward_kernel(Rows R, sb_distill d, const float* g_loss,
                                                                      int64_t g_stride, T* grad) {
    extern __shared__ uint4 dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* sh = reinterpret_cast<uint8_t*>(dyn);
    const int row_bytes = MASK == SB_MASK_NONE ? 0 : bits_bytes(R.a);
    uint8_t* sh_bits = sh + (W == 1 ? warp * row_bytes : 0);
    uint8_t* work = sh + (WARPS / W) * row_bytes + warp * GRAD_BYTES;
    const float tc = d.tail ? 1.f : R.inv_t;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        T* out = grad + row * R.a;
        const float2* s = reinterpret_cast<const float2*>(d.row_stats + 6 * row);
        const float2 st = s[0], co = s[1], te = s[2];
        const float w = g_loss[row * g_stride];
        Bits bits = {nullptr, 0};
        if (MASK != SB_MASK_NONE) {
            bits = stage<MASK, 32 * W>(sh_bits, R.mask + row * R.mask_stride, R.a, W == 1 ? lane : threadIdx.x);
            if (W == 1) __syncwarp();
            else __syncthreads();
        }
        const RowGrad r = {st.x, st.y, w * co.y, 0.f, w * co.x};
        const int2 own = grad_row<T, MASK, W, false>(x, out, bits, R.a, r, R.inv_t, work, W == 1 ? 0 : warp);
        for (int k0 = 0; k0 < d.listed; k0 += 32) {
            float v = 0.f;
            const int a = teacher<MASK>(R, d, bits, row, k0 + lane, &v);
            float q = 0.f;
            // an action that is listed again takes all of its entries' weights:
            // every one of them stores the same value, summed in the same order
            for (int j0 = 0; j0 < d.listed; j0 += 32) {
                float u = 0.f;
                const int b = j0 == k0 ? a : teacher<MASK>(R, d, bits, row, j0 + lane, &u);
                if (j0 == k0) u = v;
                const float qu = b >= 0 ? expf((u - te.x) * tc - te.y) : 0.f;
                for (int j = 0; j < 32 && j0 + j < d.listed; ++j) {
                    const int bj = __shfl_sync(ALL, b, j);
                    const float qj = __shfl_sync(ALL, qu, j);
                    if (a >= 0 && bj == a) q += qj;
                }
            }
            if (a >= 0 && a >= own.x && a < own.y)
                out[a] = from_f<T>(grad_of<false>(to_f(x[a]), r, r.l0, -w * q, R.inv_t));
        }
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

int check_rows(const sb_logits* x, Rows* R) {
    if (!x) return fail(SB_E_ARG, "logits description is NULL");
    if (x->n_rows < 0) return fail(SB_E_ARG, "n_rows < 0");
    if (x->n_actions < 1 || x->n_actions > SB_POLICY_MAX_ACTIONS)
        return fail(SB_E_ARG, "n_actions must be 1..%d, got %d", SB_POLICY_MAX_ACTIONS, x->n_actions);
    if (x->dtype != SB_DTYPE_F32 && x->dtype != SB_DTYPE_BF16 && x->dtype != SB_DTYPE_F16)
        return fail(SB_E_ARG, "bad logits dtype %d", x->dtype);
    if (x->mask_kind < SB_MASK_NONE || x->mask_kind > SB_MASK_BITS) return fail(SB_E_ARG, "bad mask kind %d", x->mask_kind);
    if (!(x->temperature > 0.f) || x->temperature == INFINITY || 1.f / x->temperature == INFINITY)
        return fail(SB_E_ARG, "temperature must be finite and > 0");
    if (x->row_stride < 0 || x->mask_stride < 0) return fail(SB_E_ARG, "negative row stride");
    if (x->n_rows == 0) return SB_OK;
    if (!x->logits || !aligned(x->logits, x->dtype == SB_DTYPE_F32 ? 4 : 2))
        return fail(SB_E_ARG, "logits NULL or not aligned to their type");
    if ((x->mask_kind != SB_MASK_NONE) != (x->mask != nullptr)) return fail(SB_E_ARG, "mask and mask_kind disagree");
    *R = {x->logits, x->mask, x->n_rows, x->row_stride, x->mask_stride, x->n_actions, 1.f / x->temperature};
    return SB_OK;
}

bool index_bytes_ok(int b) { return b == 2 || b == 4 || b == 8; }

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SB_OK : cuda_fail(e, what);
}

unsigned grid_of(int64_t rows, int w) {
    const int64_t ctas = (rows + WARPS / w - 1) / (WARPS / w);
    return (unsigned)(ctas < 0x7fffffff ? ctas : 0x7fffffff);
}

template <int V> using Const = std::integral_constant<int, V>;

// Call f(element type, mask kind, warps per row) as constants.
template <typename F>
int dispatch(const sb_logits* x, bool wide, F f) {
    auto kinds = [&](auto* t) {
        switch (x->mask_kind) {
            case SB_MASK_U8: return wide ? f(t, Const<SB_MASK_U8>{}, Const<WARPS>{}) : f(t, Const<SB_MASK_U8>{}, Const<1>{});
            case SB_MASK_BITS:
                return wide ? f(t, Const<SB_MASK_BITS>{}, Const<WARPS>{}) : f(t, Const<SB_MASK_BITS>{}, Const<1>{});
            default: return wide ? f(t, Const<SB_MASK_NONE>{}, Const<WARPS>{}) : f(t, Const<SB_MASK_NONE>{}, Const<1>{});
        }
    };
    if (x->dtype == SB_DTYPE_F32) return kinds((float*)nullptr);
    if (x->dtype == SB_DTYPE_BF16) return kinds((__nv_bfloat16*)nullptr);
    return kinds((__half*)nullptr);
}

int64_t row_bytes(const sb_logits* x) { return (int64_t)x->n_actions * (x->dtype == SB_DTYPE_F32 ? 4 : 2); }

// Four warps per row where one would have a long chain of loads for it: more
// than 4 KB of an unmasked row (32 elements a lane and turn), a mask of more
// than 16,384 actions (2 KB of staged bits a warp), or a masked gradient row
// of more than 64 KB (1 KB of zeros a turn).  Splitting a shorter masked row
// costs more than it gives: each warp pays for its own joins.
bool wide_forward(const sb_logits* x) {
    return x->mask_kind == SB_MASK_NONE ? row_bytes(x) > 4096 : x->n_actions > 16384;
}
bool wide_backward(const sb_logits* x) { return row_bytes(x) > (x->mask_kind == SB_MASK_NONE ? 4096 : 65536); }

int check_logprobs(const sb_logits* x, const sb_logprobs* o) {
    if (!o) return fail(SB_E_ARG, "outputs description is NULL");
    if (o->top < 0 || o->top > SB_POLICY_MAX_TOP) return fail(SB_E_ARG, "top must be 0..%d", SB_POLICY_MAX_TOP);
    if (o->actions && !index_bytes_ok(o->action_bytes)) return fail(SB_E_ARG, "actions must be 2, 4 or 8 bytes wide");
    if (o->actions && !aligned(o->actions, o->action_bytes)) return fail(SB_E_ARG, "actions not aligned to their type");
    return SB_OK;
}

int check_distill(const sb_logits* x, const sb_distill* d) {
    if (!d) return fail(SB_E_ARG, "teacher description is NULL");
    if (d->listed < 1 || d->listed > SB_POLICY_MAX_TEACHER)
        return fail(SB_E_ARG, "listed must be 1..%d, got %d", SB_POLICY_MAX_TEACHER, d->listed);
    if (!index_bytes_ok(d->action_bytes)) return fail(SB_E_ARG, "teacher actions must be 2, 4 or 8 bytes wide");
    if (d->teacher_dtype < SB_DTYPE_F32 || d->teacher_dtype > SB_DTYPE_F16)
        return fail(SB_E_ARG, "bad teacher dtype %d", d->teacher_dtype);
    if (d->tail != 0 && d->tail != 1) return fail(SB_E_ARG, "tail must be 0 or 1");
    if (x->n_rows == 0) return SB_OK;
    if (!d->teacher_actions || !d->teacher_logits) return fail(SB_E_ARG, "teacher actions or logits are NULL");
    if (!aligned(d->teacher_actions, d->action_bytes) ||
        !aligned(d->teacher_logits, d->teacher_dtype == SB_DTYPE_F32 ? 4 : 2))
        return fail(SB_E_ARG, "teacher actions or logits not aligned to their type");
    if (d->row_stats && !aligned(d->row_stats, 8)) return fail(SB_E_ARG, "row_stats not 8-byte aligned");
    return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

int sb_action_logprobs(const sb_logits* x, const sb_logprobs* out, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_logprobs(x, out)) != SB_OK || x->n_rows == 0) return rc;
    if (!out->entropy || (out->actions != nullptr) != (out->logprob != nullptr))
        return fail(SB_E_ARG, "entropy is NULL, or actions and logprob disagree");
    if (out->top && (!out->top_action || !out->top_logprob)) return fail(SB_E_ARG, "top outputs are NULL");
    if (out->row_stats && !aligned(out->row_stats, 8)) return fail(SB_E_ARG, "row_stats not 8-byte aligned");
    return dispatch(x, wide_forward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int smem = M == SB_MASK_NONE ? 0 : WARPS / W * bits_bytes(R.a) + WARPS * 2 * LIST;
        if (out->top)
            logprobs_kernel<T, M, W, true><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *out);
        else
            logprobs_kernel<T, M, W, false><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *out);
        return launched("logprobs_kernel launch");
    });
}

int sb_action_logprobs_backward(const sb_logits* x, const sb_logprobs* fwd, const sb_logprobs_grad* g, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_logprobs(x, fwd)) != SB_OK) return rc;
    if (!g) return fail(SB_E_ARG, "gradient description is NULL");
    if (x->n_rows == 0) return SB_OK;
    if (!g->grad || !fwd->row_stats || !fwd->entropy) return fail(SB_E_ARG, "grad, row_stats or entropy is NULL");
    if (!aligned(g->grad, x->dtype == SB_DTYPE_F32 ? 4 : 2)) return fail(SB_E_ARG, "grad not aligned to its type");
    if (!aligned(fwd->row_stats, 8)) return fail(SB_E_ARG, "row_stats not 8-byte aligned");
    if ((g->g_logprob && !fwd->actions) || (g->g_top && (!fwd->top || !fwd->top_action)))
        return fail(SB_E_ARG, "a gradient of an output that the forward call did not have");
    return dispatch(x, wide_backward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int smem = M == SB_MASK_NONE ? 0 : WARPS / W * bits_bytes(R.a) + WARPS * GRAD_BYTES;
        logprobs_backward_kernel<T, M, W><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *fwd, *g);
        return launched("logprobs_backward_kernel launch");
    });
}

int sb_distill_loss(const sb_logits* x, const sb_distill* d, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_distill(x, d)) != SB_OK || x->n_rows == 0) return rc;
    if (!d->loss) return fail(SB_E_ARG, "loss is NULL");
    return dispatch(x, wide_forward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int lists = M == SB_MASK_NONE ? 0 : WARPS * 2 * LIST;
        const int smem = WARPS / W * bits_bytes(R.a) * ((M != SB_MASK_NONE) + d->tail) + lists;
        if (d->tail)
            distill_kernel<T, M, W, true><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *d);
        else
            distill_kernel<T, M, W, false><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *d);
        return launched("distill_kernel launch");
    });
}

int sb_distill_loss_backward(const sb_logits* x, const sb_distill* d, const float* g_loss, int64_t g_loss_stride,
                             void* grad, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_distill(x, d)) != SB_OK || x->n_rows == 0) return rc;
    if (!g_loss || !grad || !d->row_stats) return fail(SB_E_ARG, "g_loss, grad or row_stats is NULL");
    if (!aligned(grad, x->dtype == SB_DTYPE_F32 ? 4 : 2)) return fail(SB_E_ARG, "grad not aligned to its type");
    return dispatch(x, wide_backward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int smem = M == SB_MASK_NONE ? 0 : WARPS / W * bits_bytes(R.a) + WARPS * GRAD_BYTES;
        distill_backward_kernel<T, M, W><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(
            R, *d, g_loss, g_loss_stride, static_cast<T*>(grad));
        return launched("distill_backward_kernel launch");
    });
}

}  // extern "C"
