// sb_policy.cuh -- what the operators on rows of policy logits under a
// legal-action mask share: log-probabilities of given actions with entropy and
// top alternatives (sb_logprobs.cu), and the divergence from a teacher's
// listed actions (sb_distill.cu), both with gradients; rows of up to 128
// actions have kernels of their own (sb_policy_small.cu).
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
// CTA where it is long (wide_forward, wide_backward).  In the forward pass that
// rule looks at the shape and the types alone, and a gradient's elements do not
// depend on who computes them.  So a row's bits do not depend on its batch nor
// on where it lies, but for rows that are read whole (no mask, or over an eighth
// legal, with more than SMALL actions): those are dealt to the lanes by sectors
// of memory, and the order of their sums goes with the row's address modulo 32
// bytes.  A legal mask is staged in shared memory as one bit per action, and only the
// logits of set bits are read: a position has some 30 legal moves of 10,000, so
// a row costs its mask and 30 sectors instead of 20 or 40 KB.  A row of which
// over an eighth is legal is read whole.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "sb_error.h"
#include "stratego_b200.h"

namespace sb {
namespace {

constexpr int WARPS = 4;                  // warps of a CTA: one row each, or one row together
constexpr unsigned ALL = 0xffffffffu;
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int LIST = 1024;                // legal actions a warp lists at once: those of 32 mask words
constexpr int WORDS = 320;                // mask words a warp looks through at once
constexpr int PASS_BYTES = 2 * (LIST + WORDS);  // shared memory of a warp's pass over a masked row
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
    // The chunk at row[first], whatever its alignment: where it is not a sector
    // of its own, from the 16-byte pieces that it touches, if those are the
    // row's (false: load it element by element).
    __device__ __forceinline__ bool load_near(const T* row, int first, int a) {
        const intptr_t p = (intptr_t)(row + first);
        if (first < 0 || first + E > a) return false;
        if ((p & 31) == 0) {
            load(row + first);
            return true;
        }
        const int off = (int)(p & 15);
        const intptr_t base = p - off;
        if (base < (intptr_t)row || base + (off ? 48 : 32) > (intptr_t)(row + a)) return false;
        const uint4* g = reinterpret_cast<const uint4*>(base);
        const uint4 x = __ldg(g), y = __ldg(g + 1), z = off ? __ldg(g + 2) : make_uint4(0, 0, 0, 0);
        uint32_t v[12] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
        if (off & 4) {
#pragma unroll
            for (int i = 0; i < 11; ++i) v[i] = v[i + 1];
        }
        if (off & 8) {
#pragma unroll
            for (int i = 0; i < 9; ++i) v[i] = v[i + 2];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * (off & 3));
        return true;
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
    __device__ __forceinline__ float max() const;  // NaN aside
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
    __half2 h;
    memcpy(&h, &w[e >> 1], 4);
    return e & 1 ? __high2float(h) : __low2float(h);
}
template <> __device__ __forceinline__ void Chunk<__half>::set(int e, float v) {
    const uint32_t b = __half_as_ushort(__float2half_rn(v));
    w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | b << 16 : (w[e >> 1] & 0xffff0000u) | b;
}

template <> __device__ __forceinline__ float Chunk<float>::max() const {
    float m = get(0);
#pragma unroll
    for (int e = 1; e < E; ++e) m = fmaxf(m, get(e));
    return fmaxf(m, NEG_INF);
}
// 16-bit elements are compared two at a time as they are.
template <> __device__ __forceinline__ float Chunk<__nv_bfloat16>::max() const {
    __nv_bfloat162 m, v;
    memcpy(&m, &w[0], 4);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        memcpy(&v, &w[i], 4);
        m = __hmax2(m, v);
    }
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), NEG_INF);
}
template <> __device__ __forceinline__ float Chunk<__half>::max() const {
    __half2 m, v;
    memcpy(&m, &w[0], 4);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        memcpy(&v, &w[i], 4);
        m = __hmax2(m, v);
    }
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), NEG_INF);
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

// Bit a + P of `w` is 1 where action a is legal.  Words past the row are 0;
// bits before it may be anything.
struct Bits {
    uint32_t* w;
    int p;
    __device__ __forceinline__ bool test(int a) const { return (w[(a + p) >> 5] >> ((a + p) & 31)) & 1; }
    // the 32 actions from 32 i on
    __device__ __forceinline__ uint32_t word(int i) const {
        const int b = 32 * i + p;
        return __funnelshift_r(w[b >> 5], w[(b >> 5) + 1], b & 31);
    }
    // `len` <= 16 bits of the actions from a on (a >= -16; 0 for those below 0)
    __device__ __forceinline__ uint32_t field(int a, int len) const {
        const int b = a + p;
        const uint32_t f = __funnelshift_r(w[b >> 5], w[(b >> 5) + 1], b & 31) & ((1u << len) - 1u);
        return a < 0 ? f & (ALL << -a) : f;
    }
};

// Bytes of a staged row: the bits, 32 of lead (16 to align a bit-packed row's
// chunks, 16 that a field below action 0 may touch) and zeros past the end.
__host__ __device__ constexpr int bits_bytes(int a) { return ((a + 7) / 8 + 32 + 48 + 15) / 16 * 16; }

__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t v) {  // bit i: byte i of v is not 0
    const uint32_t t = (((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) & 0x80808080u;
    return ((t >> 7) * 0x01020408u) >> 24 & 15u;
}

// Stage one row's mask with G threads (tid 0..G-1; the caller synchronises).
template <int MASK, int G>
__device__ __forceinline__ Bits stage(uint8_t* sh, const Rows& R, int64_t row, int tid) {
    const uint8_t* m = R.mask + row * R.mask_stride;
    const int a = R.a, h = (int)(-(intptr_t)m & 15), off = (16 - h) & 15;
    if (MASK == SB_MASK_BITS && row > 0 && row < R.n - 1 && R.mask_stride >= (a + 7) >> 3) {
        // The 16-byte chunks that the row touches, whole: the few bytes of them
        // that are not the row's belong to the rows beside it (a row here has
        // more than SMALL actions, 16 bytes).  Row byte i goes
        // to sh[16 + off + i]; the last chunk is cut off after the last action.
        const int end = 8 * off + a;  // bits from the first chunk's start
        const int last = (end - 1) >> 7;
        uint4* s4 = reinterpret_cast<uint4*>(sh + 16);
        const uint4* g4 = reinterpret_cast<const uint4*>(m - off);
#pragma unroll 3
        for (int j = tid; j < last; j += G) s4[j] = __ldg(g4 + j);
        if (tid < 2) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (tid == 0) {
                v = __ldg(g4 + last);
                const int n = end - 128 * last;  // 1..128 bits stay
                v.x &= n < 32 ? (1u << n) - 1u : ALL;
                v.y &= n < 64 ? (n > 32 ? (1u << (n - 32)) - 1u : 0u) : ALL;
                v.z &= n < 96 ? (n > 64 ? (1u << (n - 64)) - 1u : 0u) : ALL;
                v.w &= n < 128 ? (n > 96 ? (1u << (n - 96)) - 1u : 0u) : ALL;
            }
            s4[last + tid] = v;
        }
        return {reinterpret_cast<uint32_t*>(sh), 8 * (16 + off)};
    }
    if (MASK == SB_MASK_BITS) {
        // A short row, the first or the last one: the chunks inside the row, and
        // single bytes at its ends.  The row's last byte is always handled as a
        // tail byte: its bits past the last action drop.
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
    constexpr int U = 10;  // loads in flight: a row of 10,000 bytes is two turns of a warp
    for (int j0 = tid; j0 < nb; j0 += U * G) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = j0 + u * G < nb ? __ldg(g4 + j0 + u * G) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t b = 0;
            if (v[u].x | v[u].y | v[u].z | v[u].w)
                b = nonzero_bytes(v[u].x) | nonzero_bytes(v[u].y) << 4 | nonzero_bytes(v[u].z) << 8 |
                    nonzero_bytes(v[u].w) << 12;
            if (j0 + u * G < nb) s2[lead + j0 + u * G] = (uint16_t)b;
        }
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
    s.n = (float)__reduce_add_sync(ALL, (int)s.n);
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

// The legal logits of this warp's part of a row.  Two steps of compaction, as
// a position's 30 legal moves lie in some 20 of 313 mask words: the words that
// are not 0 (by ballots), then the actions of 32 such words, a lane each.  The
// actions come out in ascending order and are dealt to the lanes in turn, so
// the sums' order, and with it every bit of a listed row's result, is the same
// for any kind of mask and wherever its rows lie.  SKIP leaves out the actions of
// `skip`.  Returns how many actions were taken, or -1, none taken, for a row of
// one warp that is better read whole (pass_all): over half of its first words
// hold a legal action, and over an eighth of their actions are legal.
template <typename T, int W, bool ENT, bool TOP, bool SKIP>
__device__ __forceinline__ int pass_masked(Sum& s, Top& top, const T* x, Bits bits, Bits skip, int a, float c,
                                           uint16_t* list, int part) {
    const int lane = threadIdx.x & 31;
    const unsigned below = (1u << lane) - 1u;
    const int words = (a + 31) >> 5, per = (words + W - 1) / W;
    const int hi = W == 1 ? words : min(words, (part + 1) * per);
    uint16_t* some = list + LIST;
    auto word = [&](int i) { return SKIP ? bits.word(i) & ~skip.word(i) : bits.word(i); };
    int taken = 0;
    for (int w0 = part * per; w0 < hi; w0 += WORDS) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < WORDS / 32; ++k) {
            const int i = w0 + 32 * k + lane;
            const bool on = i < hi && word(i) != 0;
            const unsigned m = __ballot_sync(ALL, on);
            if (on) some[n + __popc(m & below)] = (uint16_t)i;
            n += __popc(m);
        }
        __syncwarp();
        if (W == 1 && !SKIP && w0 == 0 && 2 * n > min(words, WORDS)) {
            int count = 0;
            for (int j = lane; j < n; j += 32) count += __popc(word(some[j]));
            if (__reduce_add_sync(ALL, count) > 4 * min(words, WORDS)) return -1;
        }
        for (int j = 0; j < n; j += 32) {
            const int i = j + lane < n ? some[j + lane] : 0;
            uint32_t w = j + lane < n ? word(i) : 0u;
            const int count = __popc(w);
            int at = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(ALL, at, o);
                if (lane >= o) at += v;
            }
            const int total = __shfl_sync(ALL, at, 31);
            at -= count;
            while (w) {
                list[at++] = (uint16_t)(32 * i + __ffs(w) - 1);
                w &= w - 1;
            }
            __syncwarp();
            if (TOP || total <= 32) {
                for (int q = 0; q < total; q += 32) {
                    const int b = q + lane < total ? list[q + lane] : 0;
                    const float v[1] = {q + lane < total ? to_f(x[b]) : NEG_INF};
                    take<1, ENT>(s, v, c);
                    if (TOP) {
                        if (taken + q == 0) top.fill(v[0], b);
                        else top.offer(v[0], b);
                    }
                }
            } else {
                for (int q0 = 0; q0 < total; q0 += 128) {
                    float v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int b = q0 + q * 32 + lane;
                        v[q] = b < total ? to_f(x[list[b]]) : NEG_INF;
                    }
                    take<4, ENT>(s, v, c);
                }
            }
            taken += total;
            __syncwarp();
        }
    }
    return taken;
}

// ---- one pass over an unmasked row --------------------------------------------------

// A lane's own sums, with its own largest logit m as the reference (no
// exchange between lanes until the end): s = sum of exp(d), the maximum's 1
// included, t as in Sum.
struct LaneSum {
    float m, s, t;
};

// The lane's reference becomes m where that is larger.
template <bool ENT>
__device__ __forceinline__ void lane_raise(LaneSum& z, float m, float c) {
    if (m > z.m) {
        const float d = (z.m - m) * c, f = exp2_(d);
        if (ENT) z.t = f * (z.t + z.s * fmaxf(d, -1e4f));
        z.s *= f;
        z.m = m;
    }
}
template <bool ENT>
__device__ __forceinline__ void lane_add(LaneSum& z, float x, float ref, float c) {
    const float d = (x - ref) * c, e = exp2_(d);
    z.s += e;
    if (ENT) z.t = fmaf(e, fmaxf(d, -1e4f), z.t);
}

// How a warp's part of an unmasked row is dealt out: 32-byte chunks at the
// row's alignment in memory, chunk `part` * 32 + lane + n * 32 W for lane, and
// the two ends that do not fill a chunk (fewer than 32 elements) one element a
// lane of part 0.
template <typename T, int W> struct Deal {
    static constexpr int E = Chunk<T>::E;
    int head, chunks, first, end;  // `end`: the lane's element of the ends, or past the row
    __device__ __forceinline__ Deal(const T* x, int a, int part) {
        const int lane = threadIdx.x & 31;
        head = min(a, (int)((-(intptr_t)x & 31) / sizeof(T)));
        chunks = (a - head) / E;
        first = part * 32 + lane;
        end = part ? a : lane < head ? lane : chunks * E + lane;
    }
};

// Which actions of a whole row count: with F & 1 only the legal ones, with
// F & 2 not those of `skip`.
template <int F> struct Filter {
    static constexpr int kind = F;
    Bits legal, skip;
    __device__ __forceinline__ uint32_t out(int a, int len) const {
        uint32_t o = F & 1 ? ~legal.field(a, len) : 0u;
        if (F & 2) o |= skip.field(a, len);
        return o;
    }
    __device__ __forceinline__ bool has(int a) const { return !((F & 1 && !legal.test(a)) || (F & 2 && skip.test(a))); }
};

// One turn: U chunks of a lane, loaded before the first is used.
template <typename T, int W, int U, bool ENT, int F>
__device__ __forceinline__ void lane_turn(LaneSum& z, const T* body, int i, Filter<F> f, int head, float c) {
    constexpr int E = Chunk<T>::E;
    Chunk<T> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u].load(body + (i + u * 32 * W) * E);
    float m = NEG_INF;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (F) {
            const uint32_t out = f.out(head + (i + u * 32 * W) * E, E);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if ((out >> e) & 1) q[u].set(e, NEG_INF);
        }
        m = fmaxf(m, q[u].max());
    }
    lane_raise<ENT>(z, m, c);
    const float ref = z.m == NEG_INF ? 0.f : z.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) lane_add<ENT>(z, q[u].get(e), ref, c);
}

template <typename T, int W, bool ENT, int F>
__device__ __forceinline__ LaneSum pass_all(const T* x, Filter<F> f, int a, float c, int part) {
    constexpr int U = sizeof(T) == 4 ? 4 : 2;
    const Deal<T, W> deal(x, a, part);
    LaneSum z = {NEG_INF, 0.f, 0.f};
    const T* body = x + deal.head;
    const float last = deal.end < a && f.has(deal.end) ? to_f(x[deal.end]) : NEG_INF;
    int i = deal.first;
    for (; (i | 31) + (U - 1) * 32 * W < deal.chunks; i += U * 32 * W)  // while all lanes have U
        lane_turn<T, W, U, ENT, F>(z, body, i, f, deal.head, c);
    for (; i < deal.chunks; i += 32 * W) lane_turn<T, W, 1, ENT, F>(z, body, i, f, deal.head, c);
    lane_raise<ENT>(z, last, c);
    lane_add<ENT>(z, last, z.m == NEG_INF ? 0.f : z.m, c);
    return z;
}

// The lanes' sums as the row's.  Where one action holds nearly all of the mass,
// its lane goes over its own elements once more for the sum of the others.
template <typename T, int W, bool ENT, int F>
__device__ __forceinline__ Sum whole_all(LaneSum z, const T* x, Filter<F> f, int a, float c, int part, Sum* sh) {
    const float m = warp_max(z.m), d = (z.m - m) * c, w = m == NEG_INF ? 1.f : exp2_(d);
    const bool top = z.m == m && m > NEG_INF;
    Sum s = {m, top ? 1.f : 0.f, top ? z.s - 1.f : w * z.s, ENT ? w * (z.t + z.s * fmaxf(d, -1e4f)) : 0.f};
    Sum r = whole<W>(s, c, sh);
    if (r.n == 1.f && r.r < 0.015625f) {
        if (z.m == r.m) {
            constexpr int E = Chunk<T>::E;
            const Deal<T, W> deal(x, a, part);
            float rest = 0.f;
            auto add = [&](float v) { rest += v == r.m ? 0.f : exp2_((v - r.m) * c); };
            for (int i = deal.first; i < deal.chunks; i += 32 * W) {
                Chunk<T> q;
                q.load(x + deal.head + i * E);
                const uint32_t out = F ? f.out(deal.head + i * E, E) : 0u;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!(F && (out >> e) & 1)) add(q.get(e));
            }
            if (deal.end < a && f.has(deal.end)) add(to_f(x[deal.end]));
            s.r = rest;
        }
        if (W > 1) __syncthreads();
        r = whole<W>(s, c, sh);
    }
    return r;
}

// The k best of an unmasked row.  The k-th largest of the lanes' largest logits
// bounds the k-th best from below, so only the lanes that reach it look through
// their elements again (from cache), and of those only what reaches it is
// listed: k elements and a few more, in any order, which one warp then sorts.
constexpr int CANDIDATES = 512;  // for each of the row's warps

// The warp's values in descending order, lane by lane, from d0 = 1 unsorted or
// from d0 = 16 where the first half rises and the second falls.
template <int N0> __device__ __forceinline__ float sorted_down(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = N0; n <= 32; n <<= 1) {
#pragma unroll
        for (int d = n >> 1; d; d >>= 1) {
            const float o = __shfl_xor_sync(ALL, v, d);
            v = ((lane & d) == 0) == ((lane & n) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
    }
    return v;
}

// `peaks`: every warp's lanes' largest logits, sorted; returns the k-th of all.
template <int W> __device__ __forceinline__ float kth_peak(const float (*peaks)[32], int k) {
    const int lane = threadIdx.x & 31;
    float v = peaks[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v = sorted_down<32>(fmaxf(v, peaks[w][31 - lane]));
    return __shfl_sync(ALL, v, k - 1);
}

// This lane's elements of `low` and more, into cand[0 .. limit).
template <typename T, int W, int F>
__device__ __forceinline__ void list_from(float low, const T* x, Filter<F> f, int a, int part, uint64_t* cand, int limit,
                                          int* count) {
    constexpr int E = Chunk<T>::E;
    const Deal<T, W> deal(x, a, part);
    auto keep = [&](int b) {
        const int at = atomicAdd(count, 1);
        if (at < limit) cand[at] = (uint64_t)b << 32 | __float_as_uint(to_f(x[b]));
    };
    for (int i = deal.first; i < deal.chunks; i += 32 * W) {
        Chunk<T> q;
        q.load(x + deal.head + i * E);
        if (q.max() >= low) {
            uint32_t hit = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) hit |= q.get(e) >= low ? 1u << e : 0u;
            if (F) hit &= ~f.out(deal.head + i * E, E);
            for (; hit; hit &= hit - 1) keep(deal.head + i * E + __ffs(hit) - 1);
        }
    }
    if (deal.end < a && f.has(deal.end) && to_f(x[deal.end]) >= low) keep(deal.end);
}

__device__ __forceinline__ void top_of_list(Top& top, const uint64_t* cand, int n) {
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < n; i += 32) {
        const uint64_t q = i + lane < n ? cand[i + lane] : 0;
        const float v = i + lane < n ? __uint_as_float((uint32_t)q) : NEG_INF;
        if (i == 0) top.fill(v, (int)(q >> 32));
        else top.offer(v, (int)(q >> 32));
    }
}

// Where too many reach the bound (equal or sorted logits): a warp's part, all
// lanes' elements in turn.
template <typename T, int W, int F>
__device__ __forceinline__ void top_of_part(Top& top, const T* x, Filter<F> f, int a, int part) {
    constexpr int E = Chunk<T>::E;
    const Deal<T, W> deal(x, a, part);
    const int rounds = (deal.chunks + 32 * W - 1) / (32 * W) * E;
    top.offer(deal.end < a && f.has(deal.end) ? to_f(x[deal.end]) : NEG_INF, deal.end);
    for (int i = 0; i < rounds; ++i) {
        const int ch = deal.first + i / E * 32 * W, b = deal.head + ch * E + i % E;
        top.offer(ch < deal.chunks && f.has(b) ? to_f(x[b]) : NEG_INF, b);
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
// shared memory to index by.  `q`: the chunk's logits where they were loaded
// whole (`wide`).
template <typename T, bool ENT>
__device__ __forceinline__ void grad_sparse(const T* x, T* g, int first, int a, uint32_t field, bool wide, Chunk<T> q,
                                            const RowGrad& r, float inv_t, T* xs, T* gs) {
    constexpr int E = Chunk<T>::E;
    uint4* x4 = reinterpret_cast<uint4*>(xs);
    uint4* g4 = reinterpret_cast<uint4*>(gs);
    if (wide) {
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
    if (first >= 0 && first + E <= a) {
        const uint4 u = g4[0], v = g4[1];
        q.w[0] = u.x, q.w[1] = u.y, q.w[2] = u.z, q.w[3] = u.w;
        q.w[4] = v.x, q.w[5] = v.y, q.w[6] = v.z, q.w[7] = v.w;
        q.store(g + first);
    } else {
        for (int e = max(0, -first); e < E && first + e < a; ++e) g[first + e] = gs[e];
    }
}

// A chunk with every action legal.  NEAR: the logits do not lie as the gradient does.
template <typename T, bool ENT, bool NEAR>
__device__ __forceinline__ void grad_dense(const T* x, T* g, int first, int a, const RowGrad& r, float inv_t) {
    constexpr int E = Chunk<T>::E;
    Chunk<T> q;
    bool full = first >= 0 && first + E <= a;
    if (NEAR) full = q.load_near(x, first, a);
    else if (full) q.load(x + first);
    if (full) {
#pragma unroll
        for (int e = 0; e < E; ++e) q.set(e, grad_of<ENT>(q.get(e), r, r.c0, 0.f, inv_t));
        q.store(g + first);
    } else {
        for (int b = max(0, first); b < first + E && b < a; ++b)
            g[b] = from_f<T>(grad_of<ENT>(to_f(x[b]), r, r.c0, 0.f, inv_t));
    }
}

// A rest whose mass p_r the policy takes below e^-745, where 64-bit floats end,
// counts as no rest: such actions are masked inside the logits (-1e9, the
// type's lowest value), and what rounding leaves of a teacher that lists all
// the others must not be set against them.
constexpr float LOG_NO_MASS = -745.f;

// A distilled row's gradient off the listed actions, w (p Q - q_r p / p_r) / T,
// from Q and the logarithm of q_r / p_r (-inf: no rest).  The ratio itself
// leaves float32's range where the policy puts next to nothing on the rest, and
// p with it; so a ratio above 1 goes into the exponent, and what is
// exponentiated is log(q_r p / p_r) <= 0.
__device__ __forceinline__ RowGrad rest_grad(float2 stats, float total, float log_ratio, float w) {
    const float k = fmaxf(0.f, log_ratio);
    return {stats.x, stats.y - k, w * (total * expf(-k) - expf(log_ratio - k)), 0.f, 0.f};
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
        if ((((intptr_t)x ^ (intptr_t)g) & 31) == 0)
            for (int ch = lo + lane; ch < hi; ch += 32) grad_dense<T, ENT, false>(x, g, ch * E - e0, a, r, inv_t);
        else
            for (int ch = lo + lane; ch < hi; ch += 32) grad_dense<T, ENT, true>(x, g, ch * E - e0, a, r, inv_t);
    } else {
        uint32_t* list = reinterpret_cast<uint32_t*>(sh);
        T* xs = reinterpret_cast<T*>(sh + 4 * CHUNKS + lane * SLOT);
        T* gs = reinterpret_cast<T*>(sh + 4 * CHUNKS + (32 + lane) * SLOT);
        Chunk<T> zero;
        zero.fill(0);
        auto open = [&](int ch, uint32_t f) { return f != 0 || ch * E - e0 < 0 || ch * E - e0 + E > a; };
        int count = 0, from = lo;  // listed chunks; the first one whose zeros are not stored
#pragma unroll 2
        for (int c0 = lo; c0 < hi; c0 += 32) {
            const int ch = c0 + lane, to = min(c0 + 32, hi);
            const uint32_t f = ch < hi ? bits.field(ch * E - e0, E) : 0u;
            const bool put = ch < hi && open(ch, f);
            const unsigned b = __ballot_sync(ALL, put);
            if (put) list[count + __popc(b & ((1u << lane) - 1u))] = (uint32_t)ch | f << 16;
            count += __popc(b);
            if (count > CHUNKS - 32 || to == hi) {
                __syncwarp();
                // the first 32 listed chunks' logits come while the zeros go
                const uint32_t v0 = lane < count ? list[lane] : 0u;
                const int first0 = (int)(v0 & 0xffffu) * E - e0;
                const bool wide = lane < count && first0 >= 0 && first0 + E <= a && ((intptr_t)(x + first0) & 31) == 0;
                Chunk<T> q;
                if (wide) q.load(x + first0);
#pragma unroll 2
                for (int k = from + lane; k < to; k += 32)
                    if (!open(k, bits.field(k * E - e0, E))) zero.store(g + k * E - e0);
                if (lane < count) grad_sparse<T, ENT>(x, g, first0, a, v0 >> 16, wide, q, r, inv_t, xs, gs);
                if (lane + 32 < count) {  // at most CHUNKS = 64 are listed
                    const uint32_t v = list[lane + 32];
                    const int first = (int)(v & 0xffffu) * E - e0;
                    const bool too = first >= 0 && first + E <= a && ((intptr_t)(x + first) & 31) == 0;
                    if (too) q.load(x + first);
                    grad_sparse<T, ENT>(x, g, first, a, v >> 16, too, q, r, inv_t, xs, gs);
                }
                __syncwarp();
                count = 0;
                from = to;
            }
        }
    }
    __syncwarp();  // the listed actions' own values are stored over these
    return make_int2(max(0, lo * E - e0), hi * E - e0);
}

// ---- host side -----------------------------------------------------------------------------

inline int check_rows(const sb_logits* x, Rows* R) {
    if (!x) return fail(SB_E_ARG, "logits description is NULL");
    if (x->n_rows < 0) return fail(SB_E_ARG, "n_rows < 0");
    if (x->n_actions < 1 || x->n_actions > SB_POLICY_MAX_ACTIONS)
        return fail(SB_E_ARG, "n_actions must be 1..%d, got %d", SB_POLICY_MAX_ACTIONS, x->n_actions);
    if (x->dtype != SB_DTYPE_F32 && x->dtype != SB_DTYPE_BF16 && x->dtype != SB_DTYPE_F16)
        return fail(SB_E_ARG, "bad logits dtype %d", x->dtype);
    if (x->mask_kind < SB_MASK_NONE || x->mask_kind > SB_MASK_BITS) return fail(SB_E_ARG, "bad mask kind %d", x->mask_kind);
    if (!(x->temperature >= 1e-30f && x->temperature <= 1e30f))
        return fail(SB_E_ARG, "temperature must be between 1e-30 and 1e30");
    if (x->row_stride < 0 || x->mask_stride < 0) return fail(SB_E_ARG, "negative row stride");
    if (x->n_rows == 0) return SB_OK;
    if (!x->logits || !aligned(x->logits, x->dtype == SB_DTYPE_F32 ? 4 : 2))
        return fail(SB_E_ARG, "logits NULL or not aligned to their type");
    if ((x->mask_kind != SB_MASK_NONE) != (x->mask != nullptr)) return fail(SB_E_ARG, "mask and mask_kind disagree");
    *R = {x->logits, x->mask, x->n_rows, x->row_stride, x->mask_stride, x->n_actions, 1.f / x->temperature};
    return SB_OK;
}

inline bool index_bytes_ok(int b) { return b == 2 || b == 4 || b == 8; }

inline int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SB_OK : cuda_fail(e, what);
}

inline unsigned grid_of(int64_t rows, int w) {
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

inline int64_t row_bytes(const sb_logits* x) { return (int64_t)x->n_actions * (x->dtype == SB_DTYPE_F32 ? 4 : 2); }

// Four warps per row where one would have a long chain of loads for it: more
// than 4 KB of an unmasked row (32 elements a lane and turn) or a mask of more
// than 16,384 actions (2 KB of staged bits a warp).  Splitting a shorter masked
// row costs more than it gives: each warp pays for its own joins.
inline bool wide_forward(const sb_logits* x) {
    return x->mask_kind == SB_MASK_NONE ? row_bytes(x) > 4096 : x->n_actions > 16384;
}
// A gradient's elements do not depend on who computes them, so here the rows
// count too: four warps a masked row while there are fewer than 8 rows an SM
// (64 rows of 10,000 f32: 4.2 against 9.2 us; 4096 rows: 26.5 against 21.4), and
// above 64 KB a row (1 KB of zeros a turn).
inline bool wide_backward(const sb_logits* x) {
    if (x->mask_kind == SB_MASK_NONE) return row_bytes(x) > 4096;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || sm_count(dev, &sms) != SB_OK) return false;
    return row_bytes(x) > 65536 || (row_bytes(x) > 4096 && x->n_rows < 8 * (int64_t)sms);
}

}  // namespace

// Rows of up to SMALL actions: sb_policy_small.cu.
constexpr int SMALL = 128;
int small_logprobs(const sb_logits* x, const sb_logprobs& o, cudaStream_t st);
int small_logprobs_backward(const sb_logits* x, const sb_logprobs& f, const sb_logprobs_grad& g, cudaStream_t st);
int small_distill(const sb_logits* x, const sb_distill& d, cudaStream_t st);
int small_distill_backward(const sb_logits* x, const sb_distill& d, const float* g_loss, int64_t g_stride, void* grad,
                           cudaStream_t st);

}  // namespace sb
