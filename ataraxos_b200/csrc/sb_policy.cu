// sb_policy.cu -- operators on rows of policy logits under a legal-action
// mask: log-probabilities of given actions with entropy and top alternatives,
// and the divergence from a teacher's listed actions, both with gradients.
//
// Mathematics, per row with legal set L and temperature T:
//   M = max_L x, d_a = (x_a - M) / T, Z = sum_L exp(d_a), log p_a = d_a - log Z
//   entropy H = log Z - (sum_L exp(d_a) d_a) / Z
// One pass keeps (M, n, r, t): n entries equal to M, r = sum of exp(d) over
// the others, t = sum of exp(d) d.  Holding the maximum's own 1 apart from r
// keeps log Z = log n + log1p(r / n) exact to its last bits when one action
// holds nearly all of the mass.
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

constexpr int PT = 256;                   // threads of a row's CTA
constexpr unsigned ALL = 0xffffffffu;
constexpr float NEG_INF = -INFINITY;

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

template <int MASK>
__device__ __forceinline__ bool legal(const uint8_t* m, int a) {
    if (MASK == SB_MASK_U8) return m[a] != 0;
    if (MASK == SB_MASK_BITS) return (m[a >> 3] >> (a & 7)) & 1;
    return true;
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

struct Sum {
    float m, n, r, t;
};
__device__ __forceinline__ Sum empty_sum() { return {NEG_INF, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ Sum merge(Sum a, Sum b, float inv_t) {
    if (b.m > a.m) {
        const Sum c = a;
        a = b;
        b = c;
    }
    if (a.m == b.m) return {a.m, a.n + b.n, a.r + b.r, a.t + b.t};
    const float d = (b.m - a.m) * inv_t, e = expf(d), w = b.n + b.r;
    a.r += e > 0.f ? e * w : (w != w ? w : 0.f);
    if (e > 0.f) a.t += e * (b.t + w * d);
    return a;
}

__device__ __forceinline__ Sum one(float x) {
    if (x != x || x == INFINITY) return {NEG_INF, 0.f, NAN, 0.f};
    return {x, x == NEG_INF ? 0.f : 1.f, 0.f, 0.f};
}

__device__ __forceinline__ float log_z(Sum s) { return logf(s.n) + log1pf(s.r / s.n); }

__device__ Sum block_merge(Sum s, float inv_t, Sum* sh) {
    for (int o = 16; o; o >>= 1) {
        Sum b = {__shfl_xor_sync(ALL, s.m, o), __shfl_xor_sync(ALL, s.n, o), __shfl_xor_sync(ALL, s.r, o),
                 __shfl_xor_sync(ALL, s.t, o)};
        s = merge(s, b, inv_t);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    s = sh[0];
    for (int w = 1; w < PT / 32; ++w) s = merge(s, sh[w], inv_t);
    return s;
}

// (M, log Z) as the outputs and the backward pass use them: log Z = inf for a
// row without an action of non-zero probability (every p is then 0) and NaN
// for a row that holds a legal NaN or +inf.
__device__ __forceinline__ float2 stats_of(Sum s) {
    if (s.r != s.r) return make_float2(0.f, NAN);
    if (s.m == NEG_INF) return make_float2(0.f, INFINITY);
    return make_float2(s.m, log_z(s));
}

template <typename T, int MASK>
__global__ void __launch_bounds__(PT) logprobs_kernel(Rows R, sb_logprobs o) {
    __shared__ Sum sh[PT / 32];
    __shared__ float best_x[PT / 32];
    __shared__ int best_a[PT / 32];
    for (int64_t row = blockIdx.x; row < R.n; row += gridDim.x) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const uint8_t* m = R.mask + row * R.mask_stride;
        Sum s = empty_sum();
        for (int a = threadIdx.x; a < R.a; a += PT)
            if (legal<MASK>(m, a)) s = merge(s, one(to_f(x[a])), R.inv_t);
        s = block_merge(s, R.inv_t, sh);
        const float2 st = stats_of(s);
        if (threadIdx.x == 0) {
            if (o.logprob) {
                const int64_t act = load_index(o.actions, o.action_bytes, row);
                float lp = NEG_INF;
                if (act == -1) lp = 0.f;
                else if (act >= 0 && act < R.a && legal<MASK>(m, (int)act)) lp = (to_f(x[act]) - st.x) * R.inv_t - st.y;
                o.logprob[row] = lp;
            }
            o.entropy[row] = st.y == INFINITY ? 0.f : st.y - s.t / (s.n + s.r);
            if (o.row_stats) {
                o.row_stats[2 * row] = st.x;
                o.row_stats[2 * row + 1] = st.y;
            }
        }
        float last_x = INFINITY;
        int last_a = -1;
        for (int k = 0; k < o.top; ++k) {
            float bx = NEG_INF;
            int ba = -1;
            for (int a = threadIdx.x; a < R.a; a += PT) {
                if (!legal<MASK>(m, a)) continue;
                const float v = to_f(x[a]);
                if ((v < last_x || (v == last_x && a > last_a)) && v > bx) {
                    bx = v;
                    ba = a;
                }
            }
            for (int q = 16; q; q >>= 1) {
                const float vx = __shfl_xor_sync(ALL, bx, q);
                const int va = __shfl_xor_sync(ALL, ba, q);
                if (vx > bx || (vx == bx && va < ba)) {
                    bx = vx;
                    ba = va;
                }
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 0) {
                best_x[threadIdx.x >> 5] = bx;
                best_a[threadIdx.x >> 5] = ba;
            }
            __syncthreads();
            bx = best_x[0];
            ba = best_a[0];
            for (int w = 1; w < PT / 32; ++w)
                if (best_x[w] > bx || (best_x[w] == bx && best_a[w] < ba)) {
                    bx = best_x[w];
                    ba = best_a[w];
                }
            if (threadIdx.x == 0) {
                o.top_action[row * o.top + k] = ba;
                o.top_logprob[row * o.top + k] = st.y != st.y ? NAN : ba < 0 ? NEG_INF : (bx - st.x) * R.inv_t - st.y;
            }
            last_x = bx;
            last_a = ba < 0 ? 0x7fffffff : ba;
        }
    }
}

// Gradient of one row: p (c0 + c1 log p) off the listed actions, and
// p (l0 + c1 log p) + (the sum of its entries' shares) on them.
struct RowGrad {
    float m, logz, c0, c1, l0;
};

template <typename T, int MASK>
__device__ void write_grad(const Rows& R, const T* x, const uint8_t* m, T* g, RowGrad c, int listed, const int* idx,
                           const float* add) {
    for (int a = threadIdx.x; a < R.a; a += PT) {
        float v = 0.f;
        if (legal<MASK>(m, a)) {
            const float lp = (to_f(x[a]) - c.m) * R.inv_t - c.logz, p = expf(lp);
            float extra = 0.f;
            bool on = false;
            for (int k = 0; k < listed; ++k)
                if (idx[k] == a) {
                    extra += add[k];
                    on = true;
                }
            const float base = (on ? c.l0 : c.c0) + (p == 0.f ? 0.f : c.c1 * lp);
            v = (p * base + extra) * R.inv_t;
        }
        g[a] = from_f<T>(v);
    }
}

template <typename T, int MASK>
__global__ void __launch_bounds__(PT) logprobs_backward_kernel(Rows R, sb_logprobs f, sb_logprobs_grad g) {
    __shared__ int idx[SB_POLICY_MAX_TOP + 1];
    __shared__ float add[SB_POLICY_MAX_TOP + 1];
    for (int64_t row = blockIdx.x; row < R.n; row += gridDim.x) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const uint8_t* m = R.mask + row * R.mask_stride;
        __syncthreads();
        if (threadIdx.x <= f.top) {
            int64_t a = -1;
            float v = 0.f;
            if (threadIdx.x < f.top) {
                if (g.g_top) {
                    a = f.top_action[row * f.top + threadIdx.x];
                    v = g.g_top[row * f.top + threadIdx.x];
                }
            } else if (g.g_logprob) {
                a = load_index(f.actions, f.action_bytes, row);
                if (a < 0 || a >= R.a || !legal<MASK>(m, (int)a)) a = -1;
                v = g.g_logprob[row * g.g_logprob_stride];
            }
            idx[threadIdx.x] = (int)a;
            add[threadIdx.x] = a < 0 ? 0.f : v;
        }
        __syncthreads();
        float total = 0.f;
        for (int k = 0; k <= f.top; ++k) total += add[k];
        const float gh = g.g_entropy ? g.g_entropy[row * g.g_entropy_stride] : 0.f;
        RowGrad c = {f.row_stats[2 * row], f.row_stats[2 * row + 1], -(total + gh * f.entropy[row]), -gh, 0.f};
        c.l0 = c.c0;
        write_grad<T, MASK>(R, x, m, static_cast<T*>(g.grad) + row * R.a, c, f.top + 1, idx, add);
    }
}

// The kept teacher entries of a row in shared memory: idx < 0 where one is
// left out, q its weight; returns the sum of the weights.
template <int MASK>
__device__ float load_teacher(const Rows& R, const uint8_t* m, const sb_distill& d, int64_t row, int* idx, float* q,
                              Sum* sh, float* tm, float* tz) {
    __syncthreads();
    Sum s = empty_sum();
    for (int k = threadIdx.x; k < d.listed; k += PT) {
        const int64_t a = load_index(d.teacher_actions, d.action_bytes, row * d.listed + k);
        const float v = load_value(d.teacher_logits, d.teacher_dtype, row * d.listed + k);
        const bool keep = a >= 0 && a < R.a && legal<MASK>(m, (int)a) && !(v == NEG_INF);
        idx[k] = keep ? (int)a : -1;
        q[k] = v;
        if (keep) s = merge(s, one(v), R.inv_t);
    }
    *tm = 0.f;
    *tz = 0.f;
    if (!d.tail) {
        s = block_merge(s, R.inv_t, sh);
        const float2 st = stats_of(s);
        *tm = st.x;
        *tz = st.y;
    }
    __syncthreads();
    float total = 0.f;
    for (int k = 0; k < d.listed; ++k)
        if (idx[k] >= 0) total += expf((q[k] - *tm) * (d.tail ? 1.f : R.inv_t) - *tz);
    return total;
}

template <typename T, int MASK>
__global__ void __launch_bounds__(PT) distill_kernel(Rows R, sb_distill d) {
    __shared__ Sum sh[PT / 32];
    __shared__ int idx[SB_POLICY_MAX_TEACHER];
    __shared__ float val[SB_POLICY_MAX_TEACHER];
    for (int64_t row = blockIdx.x; row < R.n; row += gridDim.x) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const uint8_t* m = R.mask + row * R.mask_stride;
        float tm, tz;
        const float sq = load_teacher<MASK>(R, m, d, row, idx, val, sh, &tm, &tz);
        Sum rest = empty_sum(), in = empty_sum();
        for (int a = threadIdx.x; a < R.a; a += PT) {
            if (!legal<MASK>(m, a)) continue;
            bool on = false;
            for (int k = 0; k < d.listed; ++k) on |= idx[k] == a;
            if (on) in = merge(in, one(to_f(x[a])), R.inv_t);
            else rest = merge(rest, one(to_f(x[a])), R.inv_t);
        }
        in = block_merge(in, R.inv_t, sh);
        rest = block_merge(rest, R.inv_t, sh);
        const float2 st = stats_of(merge(in, rest, R.inv_t));
        float total = sq, loss = 0.f, share = 0.f;
        if (d.tail) {
            const bool left = rest.m > NEG_INF || rest.r != rest.r;
            const float qr = left ? fmaxf(0.f, 1.f - sq) : 0.f;
            if (qr > 0.f) {
                const float2 si = stats_of(in), sr = stats_of(rest);
                const float sp = expf((si.x - st.x) * R.inv_t + si.y - st.y);
                const float lpr = in.m == NEG_INF ? 0.f
                                  : sp < 0.5f     ? log1pf(-sp)
                                                  : (sr.x - st.x) * R.inv_t + sr.y - st.y;
                const float lqr = log1pf(-sq);
                loss = qr * (lqr - lpr);
                share = expf(lqr - lpr);
                total += qr;
            }
        }
        if (threadIdx.x == 0) {
            for (int k = 0; k < d.listed; ++k)
                if (idx[k] >= 0) {
                    const float lq = (val[k] - tm) * (d.tail ? 1.f : R.inv_t) - tz;
                    loss += expf(lq) * (lq - ((to_f(x[idx[k]]) - st.x) * R.inv_t - st.y));
                }
            d.loss[row] = loss;
            if (d.row_stats) {
                float* s = d.row_stats + 6 * row;
                s[0] = st.x;
                s[1] = st.y;
                s[2] = total;
                s[3] = total - share;
                s[4] = tm;
                s[5] = tz;
            }
        }
    }
}

template <typename T, int MASK>
__global__ void __launch_bounds__(PT) distill_backward_kernel(Rows R, sb_distill d, const float* g_loss,
                                                              int64_t g_stride, T* grad) {
    __shared__ int idx[SB_POLICY_MAX_TEACHER];
    __shared__ float add[SB_POLICY_MAX_TEACHER];
    for (int64_t row = blockIdx.x; row < R.n; row += gridDim.x) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const uint8_t* m = R.mask + row * R.mask_stride;
        const float* s = d.row_stats + 6 * row;
        const float w = g_loss[row * g_stride];
        __syncthreads();
        for (int k = threadIdx.x; k < d.listed; k += PT) {
            const int64_t a = load_index(d.teacher_actions, d.action_bytes, row * d.listed + k);
            const float v = load_value(d.teacher_logits, d.teacher_dtype, row * d.listed + k);
            const bool keep = a >= 0 && a < R.a && legal<MASK>(m, (int)a) && !(v == NEG_INF);
            idx[k] = keep ? (int)a : -1;
            add[k] = -w * expf((v - s[4]) * (d.tail ? 1.f : R.inv_t) - s[5]);
        }
        __syncthreads();
        RowGrad c = {s[0], s[1], w * s[3], 0.f, w * s[2]};
        write_grad<T, MASK>(R, x, m, grad + row * R.a, c, d.listed, idx, add);
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

unsigned grid_of(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

// Call f with the logits' element type and the mask kind as constants.
template <typename F>
int dispatch(const sb_logits* x, F f) {
#define SB_KINDS(T)                                                                                     \
    switch (x->mask_kind) {                                                                             \
        case SB_MASK_U8: return f((T*)nullptr, std::integral_constant<int, SB_MASK_U8>{});              \
        case SB_MASK_BITS: return f((T*)nullptr, std::integral_constant<int, SB_MASK_BITS>{});          \
        default: return f((T*)nullptr, std::integral_constant<int, SB_MASK_NONE>{});                    \
    }
    if (x->dtype == SB_DTYPE_F32) SB_KINDS(float)
    if (x->dtype == SB_DTYPE_BF16) SB_KINDS(__nv_bfloat16)
    SB_KINDS(__half)
#undef SB_KINDS
}

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
    return dispatch(x, [&](auto* t, auto mask) {
        using T = std::remove_pointer_t<decltype(t)>;
        logprobs_kernel<T, decltype(mask)::value><<<grid_of(R.n), PT, 0, (cudaStream_t)stream>>>(R, *out);
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
    if ((g->g_logprob && !fwd->actions) || (g->g_top && (!fwd->top || !fwd->top_action)))
        return fail(SB_E_ARG, "a gradient of an output that the forward call did not have");
    return dispatch(x, [&](auto* t, auto mask) {
        using T = std::remove_pointer_t<decltype(t)>;
        logprobs_backward_kernel<T, decltype(mask)::value><<<grid_of(R.n), PT, 0, (cudaStream_t)stream>>>(R, *fwd, *g);
        return launched("logprobs_backward_kernel launch");
    });
}

int sb_distill_loss(const sb_logits* x, const sb_distill* d, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_distill(x, d)) != SB_OK || x->n_rows == 0) return rc;
    if (!d->loss) return fail(SB_E_ARG, "loss is NULL");
    return dispatch(x, [&](auto* t, auto mask) {
        using T = std::remove_pointer_t<decltype(t)>;
        distill_kernel<T, decltype(mask)::value><<<grid_of(R.n), PT, 0, (cudaStream_t)stream>>>(R, *d);
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
    return dispatch(x, [&](auto* t, auto mask) {
        using T = std::remove_pointer_t<decltype(t)>;
        distill_backward_kernel<T, decltype(mask)::value><<<grid_of(R.n), PT, 0, (cudaStream_t)stream>>>(
            R, *d, g_loss, g_loss_stride, static_cast<T*>(grad));
        return launched("distill_backward_kernel launch");
    });
}

}  // extern "C"
