// sb_policy_small.cu -- the policy operators on rows of up to 128 actions (a
// head over squares, piece types, setup slots).
//
// Eight lanes share a row, four rows a warp, and lane l holds actions
// l, l + 8, l + 16, ... in registers: a reduction is three exchanges for four
// rows together, and one byte of a bit-packed mask serves the eight lanes of a
// turn.  Loads are one element wide, so rows may lie at any stride or
// offset; the lanes of a row read neighbouring elements.  A gradient is put
// together in shared memory and stored as the contiguous block that four rows
// are.  The kernels are bound by their instructions (200,003 rows of 100 f16
// logits: log-probabilities 91 a row forward in 29 us, 175 back in 39 us,
// against 7 and 13 us of bytes; distillation of 16 listed with tail 56 and 65 us
// against 12 and 19), so the actions of a lane are a constant, and by latency:
// the CTAs per SM of their launch bounds were the fastest of 6 to 12, although the
// forward kernels of 13 and 16 actions a lane spill some registers for them (48 to
// 148 bytes read back in distillation, 40 in log-probabilities of 16).
#include "sb_policy.cuh"

namespace sb {
namespace {

constexpr int G = 8;             // lanes of a row
constexpr int RW = 32 / G;       // rows of a warp

__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(ALL, v, o));
    return v;
}
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}

// One lane's actions of a row: their logits (-inf where not legal) and bit i
// for a legal l + 8 i.  NI: actions of a lane, at least ceil(A / 8).
template <int NI> struct Part {
    float v[NI];
    uint32_t ok;
};

template <typename T, int NI>
__device__ __forceinline__ Part<NI> load_part(const Rows& R, int kind, int64_t row, bool live, int l) {
    Part<NI> p;
    p.ok = 0;
    const T* x = static_cast<const T*>(R.x) + row * R.stride + l;
    const uint8_t* m = R.mask + row * R.mask_stride;
    const int n = live ? (R.a - l + G - 1) / G : 0;
    if (kind == SB_MASK_NONE) {
        p.ok = n > 0 ? (1u << n) - 1u : 0u;
    } else if (kind == SB_MASK_U8) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (i < n && m[l + G * i]) p.ok |= 1u << i;
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (i < n) p.ok |= ((m[i] >> l) & 1u) << i;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) p.v[i] = (p.ok >> i) & 1 ? to_f(x[G * i]) : NEG_INF;
    return p;
}

// The row's sum, in all of its lanes, over the lane's actions in `ok` (ALL: of
// all, as the others are -inf already).  The maximum's own 1 is taken off the
// lanes' sums at the end, or left out of them one by one where it is nearly
// all of the mass.
template <bool ENT, int NI>
__device__ __forceinline__ Sum sum_part(const Part<NI>& p, uint32_t ok, float c) {
    auto at = [&](int i) { return ok == ALL || (ok >> i) & 1 ? p.v[i] : NEG_INF; };
    Sum s = no_sum();
#pragma unroll
    for (int i = 0; i < NI; ++i) s.m = fmaxf(s.m, at(i));
    const float mine = s.m;
    s.m = group_max(mine);
    const float ref = s.m == NEG_INF ? 0.f : s.m;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const float d = (at(i) - ref) * c, e = exp2_(d);
        s.r += e;
        if (ENT) s.t = fmaf(e, fmaxf(d, -1e4f), s.t);
    }
    const bool top = mine == s.m && s.m > NEG_INF;
    const float all = s.r;
    s.n = group_sum(top ? 1.f : 0.f);
    s.r = group_sum(top ? all - 1.f : all);
    if (ENT) s.t = group_sum(s.t);
    if (__any_sync(ALL, s.n == 1.f && s.r < 0.015625f)) {
        float rest = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) rest += at(i) == ref ? 0.f : exp2_((at(i) - ref) * c);
        rest = group_sum(rest);
        if (s.n == 1.f && s.r < 0.015625f) s.r = rest;
    }
    return s;
}

// Whether action a (any integer) is legal in this lane's row.
__device__ __forceinline__ bool legal_in(uint32_t ok, int64_t a, int actions) {
    const bool in = a >= 0 && a < actions;
    const int b = in ? (int)a : 0;
    return ((__shfl_sync(ALL, ok, b % G, G) >> (b / G)) & 1) && in;
}

template <typename T, int NI>
__global__ void __launch_bounds__(WARPS * 32, 10) small_logprobs_kernel(Rows R, int kind, sb_logprobs o) {
    const int lane = threadIdx.x & 31, l = lane % G;
    const float c = R.inv_t * LOG2E;
    const int64_t step = (int64_t)gridDim.x * (WARPS * RW);
    for (int64_t row0 = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * RW; row0 < R.n; row0 += step) {
        const int64_t row = row0 + lane / G;
        const bool live = row < R.n;
        int64_t act = -1;
        if (live && o.actions) act = load_index(o.actions, o.action_bytes, row);
        const bool in = act >= 0 && act < R.a;
        const float xa = in ? to_f(static_cast<const T*>(R.x)[row * R.stride + act]) : 0.f;
        const Part<NI> p = load_part<T, NI>(R, kind, row, live, l);
        const bool legal = legal_in(p.ok, act, R.a);
        const Sum s = sum_part<true>(p, ALL, c);
        const float2 st = stats_of(s);
        if (live && l == 0) {
            if (o.logprob) o.logprob[row] = act == -1 ? 0.f : legal ? (xa - st.x) * R.inv_t - st.y : NEG_INF;
            o.entropy[row] = st.y == INFINITY ? 0.f : st.y - LN2 * s.t / (s.n + s.r);
            if (o.row_stats) *reinterpret_cast<float2*>(o.row_stats + 2 * row) = st;
        }
        uint32_t left = p.ok;
        for (int k = 0; k < o.top; ++k) {  // the best of what is left, ties to the lower action
            float bx = NEG_INF;
            int ba = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (((left >> i) & 1) && p.v[i] > bx) {
                    bx = p.v[i];
                    ba = l + G * i;
                }
#pragma unroll
            for (int q = G / 2; q; q >>= 1) {
                const float ox = __shfl_xor_sync(ALL, bx, q);
                const int oa = __shfl_xor_sync(ALL, ba, q);
                if (ox > bx || (ox == bx && oa < ba)) {
                    bx = ox;
                    ba = oa;
                }
            }
            const bool some = bx > NEG_INF;
            if (some && ba % G == l) left &= ~(1u << (ba / G));
            if (live && l == k % G) {
                o.top_action[row * o.top + k] = some ? ba : -1;
                o.top_logprob[row * o.top + k] = st.y != st.y ? NAN : some ? (bx - st.x) * R.inv_t - st.y : NEG_INF;
            }
        }
    }
}

// A warp's four gradient rows from shared memory to where they lie side by side.
template <typename T>
__device__ __forceinline__ void store_rows(const T* sh, T* out, int a, int64_t rows) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (rows >= RW && ((intptr_t)out & 7) == 0) {  // four rows are a multiple of 8 bytes
        const uint2* s = reinterpret_cast<const uint2*>(sh);
        uint2* g = reinterpret_cast<uint2*>(out);
        for (int i = lane; i < RW * a * (int)sizeof(T) / 8; i += 32) g[i] = s[i];
    } else {
        const int n = (int)(rows < RW ? rows : RW) * a;
        for (int i = lane; i < n; i += 32) out[i] = sh[i];
    }
    __syncwarp();
}

template <typename T, int NI>
__global__ void __launch_bounds__(WARPS * 32, 8) small_logprobs_backward_kernel(Rows R, int kind, sb_logprobs f,
                                                                             sb_logprobs_grad g) {
    __shared__ __align__(16) T rows[WARPS][RW * SMALL];
    __shared__ float adds[WARPS][RW][SMALL];
    const int lane = threadIdx.x & 31, l = lane % G, q = lane / G;
    T* sh = rows[threadIdx.x >> 5];
    float* add = adds[threadIdx.x >> 5][q];
    const int64_t step = (int64_t)gridDim.x * (WARPS * RW);
    for (int64_t row0 = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * RW; row0 < R.n; row0 += step) {
        const int64_t row = row0 + q;
        const bool live = row < R.n;
        int64_t act = -1;
        float ga = 0.f, gh = 0.f, h = 0.f;
        float2 st = make_float2(0.f, INFINITY);
        if (live) {
            if (g.g_logprob) {
                act = load_index(f.actions, f.action_bytes, row);
                ga = g.g_logprob[row * g.g_logprob_stride];
            }
            if (g.g_entropy) gh = g.g_entropy[row * g.g_entropy_stride];
            st = *reinterpret_cast<const float2*>(f.row_stats + 2 * row);
            h = f.entropy[row];
        }
        const Part<NI> p = load_part<T, NI>(R, kind, row, live, l);
        if (!legal_in(p.ok, act, R.a)) {
            act = -1;
            ga = 0.f;
        }
        const int mine = act >= 0 && (int)act % G == l ? (int)act / G : -1;  // the given action, if it is the lane's
        float total = ga;
        if (g.g_top) {  // the alternatives are all different actions
            for (int i = l; i < R.a; i += G) add[i] = 0.f;
            __syncwarp();
            float shares = 0.f;
            for (int k = l; live && k < f.top; k += G) {
                const int64_t a = f.top_action[row * f.top + k];
                if (a >= 0 && a < R.a) {
                    add[a] = g.g_top[row * f.top + k];
                    shares += add[a];
                }
            }
            total += group_sum(shares);
            __syncwarp();
        }
        const RowGrad r = {st.x, st.y, -(total + gh * h), -gh, 0.f};
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int a = l + G * i;
            if (a < R.a) {
                const float e = (i == mine ? ga : 0.f) + (g.g_top ? add[a] : 0.f);
                sh[q * R.a + a] = from_f<T>((p.ok >> i) & 1 ? grad_of<true>(p.v[i], r, r.c0, e, R.inv_t) : 0.f);
            }
        }
        store_rows(sh, static_cast<T*>(g.grad) + row0 * R.a, R.a, R.n - row0);
    }
}

// Teacher entry k of a row (the same round in all lanes): its action, -1 where it is left out.
__device__ __forceinline__ int small_teacher(const Rows& R, const sb_distill& d, uint32_t ok, int64_t row, bool live,
                                             int k, float* v) {
    int64_t a = -1;
    *v = NEG_INF;
    if (live && k < d.listed) {
        a = load_index(d.teacher_actions, d.action_bytes, row * d.listed + k);
        *v = load_value(d.teacher_logits, d.teacher_dtype, row * d.listed + k);
    }
    return legal_in(ok, a, R.a) && !(*v == NEG_INF) ? (int)a : -1;
}

template <typename T, int NI>
__global__ void __launch_bounds__(WARPS * 32, 10) small_distill_kernel(Rows R, int kind, sb_distill d) {
    const int lane = threadIdx.x & 31, l = lane % G;
    const float c = R.inv_t * LOG2E, tc = d.tail ? 1.f : R.inv_t;
    const int64_t step = (int64_t)gridDim.x * (WARPS * RW);
    for (int64_t row0 = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * RW; row0 < R.n; row0 += step) {
        const int64_t row = row0 + lane / G;
        const bool live = row < R.n;
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const Part<NI> p = load_part<T, NI>(R, kind, row, live, l);
        const float2 st = stats_of(sum_part<false>(p, ALL, c));
        float2 tst = make_float2(0.f, 0.f);
        if (!d.tail) {
            float m = NEG_INF;
            for (int k = l; k < (d.listed + G - 1) / G * G; k += G) {
                float v;
                if (small_teacher(R, d, p.ok, row, live, k, &v) >= 0) m = fmaxf(m, v);
            }
            m = group_max(m);
            Sum s = {m, 0.f, 0.f, 0.f};
            for (int k = l; k < (d.listed + G - 1) / G * G; k += G) {
                float v;
                if (small_teacher(R, d, p.ok, row, live, k, &v) >= 0) {
                    if (v == m) s.n += 1.f;
                    else s.r += exp2_((v - (m == NEG_INF ? 0.f : m)) * c);
                }
            }
            s.n = group_sum(s.n);
            s.r = group_sum(s.r);
            tst = stats_of(s);
        }
        float loss = 0.f, total = 0.f, log_ratio = NEG_INF;
        uint32_t listed = 0;  // bit i: the lane's action l + 8 i is listed
        for (int k = l; k < (d.listed + G - 1) / G * G; k += G) {
            float v;
            const int a = small_teacher(R, d, p.ok, row, live, k, &v);
            if (a >= 0) {
                const float lq = (v - tst.x) * tc - tst.y, q = expf(lq);
                if (q > 0.f || q != q) loss += q * (lq - ((to_f(x[a]) - st.x) * R.inv_t - st.y));
                total += q;
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const int b = __shfl_sync(ALL, a, j, G);
                if (b >= 0 && b % G == l) listed |= 1u << (b / G);
            }
        }
        loss = group_sum(loss);
        total = group_sum(total);
        const uint32_t rest = p.ok & ~listed;
        const bool some = (__ballot_sync(ALL, rest != 0) >> (lane & ~(G - 1)) & ((1u << G) - 1u)) != 0;
        const float qr = d.tail && some ? fmaxf(0.f, 1.f - total) : 0.f;
        if (__any_sync(ALL, qr > 0.f)) {
            float sp = 0.f;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if ((listed >> i) & 1) sp += exp2_(((p.v[i] - st.x) * R.inv_t - st.y) * LOG2E);
            sp = group_sum(sp);
            const Sum s = sum_part<false>(p, rest, c);
            const float2 sr = stats_of(s);
            const float lpr = sp < 0.5f          ? log1pf(-sp)
                              : s.m > NEG_INF ? (sr.x - st.x) * R.inv_t + sr.y - st.y
                                              : NEG_INF;
            if (qr > 0.f && lpr > LOG_NO_MASS) {
                const float lqr = log1pf(-total);
                loss += qr * (lqr - lpr);
                log_ratio = lqr - lpr;
                total += qr;
            }
        }
        if (live && l == 0) {
            d.loss[row] = st.y != st.y ? NAN : loss;  // a spoiled row's, whatever is kept
            if (d.row_stats) {
                float2* o = reinterpret_cast<float2*>(d.row_stats + 6 * row);
                o[0] = st;
                o[1] = make_float2(total, log_ratio);
                o[2] = tst;
            }
        }
    }
}

template <typename T, int NI>
__global__ void __launch_bounds__(WARPS * 32, 8) small_distill_backward_kernel(Rows R, int kind, sb_distill d,
                                                                            const float* g_loss, int64_t g_stride, T* grad) {
    __shared__ __align__(16) T rows[WARPS][RW * SMALL];
    __shared__ float weights[WARPS][RW][SMALL];
    const int lane = threadIdx.x & 31, l = lane % G, q = lane / G;
    T* sh = rows[threadIdx.x >> 5];
    float* wt = weights[threadIdx.x >> 5][q];
    const float tc = d.tail ? 1.f : R.inv_t;
    const int64_t step = (int64_t)gridDim.x * (WARPS * RW);
    for (int64_t row0 = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * RW; row0 < R.n; row0 += step) {
        const int64_t row = row0 + q;
        const bool live = row < R.n;
        float2 st = make_float2(0.f, INFINITY), co = make_float2(0.f, 0.f), te = co;
        float w = 0.f;
        if (live) {
            const float2* s = reinterpret_cast<const float2*>(d.row_stats + 6 * row);
            st = s[0], co = s[1], te = s[2];
            w = g_loss[row * g_stride];
        }
        const Part<NI> p = load_part<T, NI>(R, kind, row, live, l);
        for (int i = l; i < R.a; i += G) wt[i] = 0.f;
        uint32_t listed = 0;
        for (int k = l; k < (d.listed + G - 1) / G * G; k += G) {
            float v;
            const int a = small_teacher(R, d, p.ok, row, live, k, &v);
            const float qk = a >= 0 ? expf((v - te.x) * tc - te.y) : 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {  // an action listed again adds up, in the entries' order
                const int b = __shfl_sync(ALL, a, j, G);
                const float qj = __shfl_sync(ALL, qk, j, G);
                if (b >= 0 && b % G == l) {
                    wt[b] += qj;
                    listed |= 1u << (b / G);
                }
            }
        }
        const RowGrad r = {st.x, st.y, 0.f, 0.f, w * co.x}, rest = rest_grad(st, co.x, co.y, w);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int a = l + G * i;
            if (a < R.a) {
                const bool on = (listed >> i) & 1;
                const float e = on ? -w * wt[a] : 0.f;
                const RowGrad s = {r.m, on ? r.logz : rest.logz, 0.f, 0.f, 0.f};
                sh[q * R.a + a] =
                    from_f<T>((p.ok >> i) & 1 ? grad_of<false>(p.v[i], s, on ? r.l0 : rest.c0, e, R.inv_t) : 0.f);
            }
        }
        store_rows(sh, grad + row0 * R.a, R.a, R.n - row0);
    }
}

Rows rows_of(const sb_logits* x) {
    return {x->logits, x->mask, x->n_rows, x->row_stride, x->mask_stride, x->n_actions, 1.f / x->temperature};
}

unsigned small_grid(int64_t rows) { return grid_of(rows, 1) > 4 ? (grid_of(rows, 1) + RW - 1) / RW : 1; }

// Call f(element type, actions of a lane) as constants.
template <typename F>
int by_type(const sb_logits* x, F f) {
    auto sizes = [&](auto* t) {
        const int n = (x->n_actions + G - 1) / G;
        if (n <= 4) return f(t, std::integral_constant<int, 4>{});
        if (n <= 8) return f(t, std::integral_constant<int, 8>{});
        if (n <= 13) return f(t, std::integral_constant<int, 13>{});
        return f(t, std::integral_constant<int, SMALL / G>{});
    };
    if (x->dtype == SB_DTYPE_F32) return sizes((float*)nullptr);
    if (x->dtype == SB_DTYPE_BF16) return sizes((__nv_bfloat16*)nullptr);
    return sizes((__half*)nullptr);
}

}  // namespace

int small_logprobs(const sb_logits* x, const sb_logprobs& o, cudaStream_t st) {
    return by_type(x, [&](auto* t, auto ni) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int NI = decltype(ni)::value;
        small_logprobs_kernel<T, NI><<<small_grid(x->n_rows), WARPS * 32, 0, st>>>(rows_of(x), x->mask_kind, o);
        return launched("small_logprobs_kernel launch");
    });
}

int small_logprobs_backward(const sb_logits* x, const sb_logprobs& f, const sb_logprobs_grad& g, cudaStream_t st) {
    return by_type(x, [&](auto* t, auto ni) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int NI = decltype(ni)::value;
        small_logprobs_backward_kernel<T, NI><<<small_grid(x->n_rows), WARPS * 32, 0, st>>>(rows_of(x), x->mask_kind, f, g);
        return launched("small_logprobs_backward_kernel launch");
    });
}

int small_distill(const sb_logits* x, const sb_distill& d, cudaStream_t st) {
    return by_type(x, [&](auto* t, auto ni) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int NI = decltype(ni)::value;
        small_distill_kernel<T, NI><<<small_grid(x->n_rows), WARPS * 32, 0, st>>>(rows_of(x), x->mask_kind, d);
        return launched("small_distill_kernel launch");
    });
}

int small_distill_backward(const sb_logits* x, const sb_distill& d, const float* g_loss, int64_t g_stride, void* grad,
                           cudaStream_t st) {
    return by_type(x, [&](auto* t, auto ni) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int NI = decltype(ni)::value;
        small_distill_backward_kernel<T, NI><<<small_grid(x->n_rows), WARPS * 32, 0, st>>>(rows_of(x), x->mask_kind, d, g_loss,
                                                                                      g_stride, static_cast<T*>(grad));
        return launched("small_distill_backward_kernel launch");
    });
}

}  // namespace sb
