// sb_distill.cu -- divergence of policy rows from a teacher's listed actions, and
// its gradient.
#include "sb_policy.cuh"

namespace sb {
namespace {

// ---- distillation ------------------------------------------------------------------------

// Kept per row for the backward pass: (M, log Z), (Q, log(q_r / p_r)) and the
// teacher's own (maximum, log sum).

// This lane's teacher entry of a round of 32: its action (-1 where it is left
// out), logit and student logit.  The first round is loaded beside the mask
// and looked at when that has come: a warp that waits for an action issues no
// other load.
struct Entry {
    int a;
    float v, x;
};
struct Raw {
    int64_t a;
    float v;
};
__device__ __forceinline__ Raw load_raw(const sb_distill& d, int64_t row, int k) {
    if (k >= d.listed) return {-1, NEG_INF};
    return {load_index(d.teacher_actions, d.action_bytes, row * d.listed + k),
            load_value(d.teacher_logits, d.teacher_dtype, row * d.listed + k)};
}
template <typename T, int MASK>
__device__ __forceinline__ Entry entry_of(const Rows& R, const T* x, Bits bits, Raw q) {
    Entry e = {-1, q.v, 0.f};
    if (q.a >= 0 && q.a < R.a && !(q.v == NEG_INF) && (MASK == SB_MASK_NONE || bits.test((int)q.a))) {
        e.a = (int)q.a;
        e.x = to_f(x[q.a]);
    }
    return e;
}

// Loss (32,768 bf16 rows, bit masks, 32 listed, tail: 49 us; 4096 unmasked f16
// rows 22.4 us, 82 MB at 3.7 TB/s): one pass for the row's (M, Z), then the
// teacher's entries by one warp.  With the tail, the unlisted actions' own mass
// p_r is 1 - sum p while that keeps its digits (sum p < 1/2), nothing where every
// legal action is listed, and otherwise summed by a second pass that leaves the
// listed ones out.
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
    uint16_t* list = reinterpret_cast<uint16_t*>(sh + (WARPS / W) * row_bytes + warp * PASS_BYTES);
    const float c = R.inv_t * LOG2E, tc = TAIL ? 1.f : R.inv_t;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        const Raw raw = load_raw(d, row, lane);
        Bits bits = {nullptr, 0};
        if (MASK != SB_MASK_NONE) bits = stage<MASK, 32 * W>(sh_bits, R, row, tid);
        // which actions are listed, as bits: needed at once to find an entry's
        // action in an earlier round, else only for a second pass
        const bool rounds = TAIL && d.listed > 32;
        auto clear = [&] {
            for (int i = tid; i < bits_bytes(R.a) / 4; i += 32 * W) sh_skip[i] = 0;
        };
        if (rounds) clear();
        if (W == 1) __syncwarp();
        else __syncthreads();
        const Bits skip = {sh_skip, bits.p};
        const Entry e0 = entry_of<T, MASK>(R, x, bits, raw);
        auto entry = [&](int k0) { return k0 ? entry_of<T, MASK>(R, x, bits, load_raw(d, row, k0 + lane)) : e0; };
        Sum s = no_sum();
        Top none;
        int legal = 0;
        bool dense = MASK == SB_MASK_NONE;
        auto read_whole = [&](auto f) {
            constexpr int F = decltype(f)::kind;
            return whole_all<T, W, false, F>(pass_all<T, W, false, F>(x, f, R.a, c, part), x, f, R.a, c, part, sums);
        };
        if (MASK == SB_MASK_NONE) {
            s = read_whole(Filter<0>{});
            legal = R.a;
        } else {
            legal = pass_masked<T, W, false, false, false>(s, none, x, bits, bits, R.a, c, list, part);
            if (W > 1) {
                if (lane == 0) counts[warp] = legal;
                s = whole<W>(s, c, sums);
                legal = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) legal += counts[w];
            } else if (legal < 0) {
                dense = true;
                s = read_whole(Filter<1>{bits, bits});
                int mine = 0;
                for (int i = lane; i < (R.a + 31) >> 5; i += 32) mine += __popc(bits.word(i));
                legal = __reduce_add_sync(ALL, mine);
            } else {
                s = whole<W>(s, c, sums);
            }
        }
        const float2 st = stats_of(s);
        float loss = 0.f, total = 0.f, log_ratio = NEG_INF;
        float2 tst = make_float2(0.f, 0.f);
        bool more = false;  // a second pass is needed
        bool lead0 = false;  // entry e0 is its action's first
        if (W == 1 || warp == 0) {
            if (!TAIL) {
                Sum ts = no_sum();
                for (int k0 = 0; k0 < d.listed; k0 += 32) {
                    const Entry e = entry(k0);
                    const float t[1] = {e.a >= 0 ? e.v : NEG_INF};
                    take<1, false>(ts, t, c);
                }
                tst = stats_of(whole<1>(ts, c, nullptr));
            }
            float sp = 0.f;
            int unique = 0;
            for (int k0 = 0; k0 < d.listed; k0 += 32) {
                const Entry e = entry(k0);
                const int a = e.a;
                float p = 0.f;
                if (a >= 0) {
                    const float lq = (e.v - tst.x) * tc - tst.y, q = expf(lq), lp = (e.x - st.x) * R.inv_t - st.y;
                    loss += q > 0.f || q != q ? q * (lq - lp) : 0.f;
                    total += q;
                    p = expf(lp);
                }
                if (TAIL) {  // an action's first entry stands for it in p
                    const unsigned peers = __match_any_sync(ALL, a);
                    bool lead = a >= 0 && (peers & ((1u << lane) - 1u)) == 0;
                    if (rounds) {
                        lead = lead && !skip.test(a);
                        __syncwarp();
                        if (lead) atomicOr(&sh_skip[(a + skip.p) >> 5], 1u << ((a + skip.p) & 31));
                        __syncwarp();
                    }
                    if (lead) sp += p;
                    if (k0 == 0) lead0 = lead;
                    unique += __popc(__ballot_sync(ALL, lead));
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
                    log_ratio = lqr - lpr;
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
                if (!rounds) {
                    clear();
                    if (W == 1) __syncwarp();
                    else __syncthreads();
                    if (lead0) atomicOr(&sh_skip[(e0.a + skip.p) >> 5], 1u << ((e0.a + skip.p) & 31));
                    if (W == 1) __syncwarp();
                    else __syncthreads();
                }
                Sum rest = no_sum();
                if (MASK == SB_MASK_NONE) {
                    rest = read_whole(Filter<2>{skip, skip});
                } else if (W == 1 && dense) {
                    rest = read_whole(Filter<3>{bits, skip});
                } else {
                    pass_masked<T, W, false, false, true>(rest, none, x, bits, skip, R.a, c, list, part);
                    rest = whole<W>(rest, c, sums);
                }
                const float2 sr = stats_of(rest);
                const float lpr = rest.m > NEG_INF ? (sr.x - st.x) * R.inv_t + sr.y - st.y : NEG_INF;
                if ((W == 1 || warp == 0) && lpr > LOG_NO_MASS) {
                    const float qr = fmaxf(0.f, 1.f - total), lqr = log1pf(-total);
                    loss += qr * (lqr - lpr);
                    log_ratio = lqr - lpr;
                    total += qr;
                }
            }
        }
        if ((W == 1 || warp == 0) && lane == 0) {
            d.loss[row] = st.y != st.y ? NAN : loss;  // a spoiled row's, whatever is kept
            if (d.row_stats) {
                float2* o = reinterpret_cast<float2*>(d.row_stats + 6 * row);
                o[0] = st;
                o[1] = make_float2(total, log_ratio);
                o[2] = tst;
            }
        }
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

// Every row as p (Q - q_r / p_r), then the listed actions' own values over it.
// Bound by the gradient's bytes: 32,768 bf16 rows 140 us (0.74 GB, 5.3 TB/s).
// Above 32 listed every group of 32 walks all entries for repeats, which grows
// with the square: 4096 bf16 rows under bit masks, forward and back together, 28
// us at 32 listed, 37 at 64, 61 at 128, 513 at 512 (unmasked: 52, 74, 164, 1870).
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
        const Raw raw = load_raw(d, row, lane);
        Bits bits = {nullptr, 0};
        if (MASK != SB_MASK_NONE) {
            bits = stage<MASK, 32 * W>(sh_bits, R, row, W == 1 ? lane : threadIdx.x);
            if (W == 1) __syncwarp();
            else __syncthreads();
        }
        auto entry = [&](int k0) { return entry_of<T, MASK>(R, x, bits, load_raw(d, row, k0 + lane)); };
        const Entry e0 = entry_of<T, MASK>(R, x, bits, raw);
        const RowGrad r = {st.x, st.y, 0.f, 0.f, w * co.x};  // of the listed actions
        const int2 own = grad_row<T, MASK, W, false>(x, out, bits, R.a, rest_grad(st, co.x, co.y, w), R.inv_t, work,
                                                   W == 1 ? 0 : warp);
        for (int k0 = 0; k0 < d.listed; k0 += 32) {
            const Entry e = k0 ? entry(k0) : e0;
            float q = e.a >= 0 ? expf((e.v - te.x) * tc - te.y) : 0.f;
            // An action that is listed again takes all of its entries' weights:
            // each of its lanes adds them in the entries' order and stores the
            // same value.
            const unsigned peers = __match_any_sync(ALL, e.a);
            if (d.listed > 32 || __any_sync(ALL, e.a >= 0 && (peers & (peers - 1)))) {
                q = 0.f;
                for (int j0 = 0; j0 < d.listed; j0 += 32) {
                    const Entry f = j0 == k0 ? e : entry(j0);
                    const float qf = f.a >= 0 ? expf((f.v - te.x) * tc - te.y) : 0.f;
                    for (int j = 0; j < 32 && j0 + j < d.listed; ++j) {
                        const int b = __shfl_sync(ALL, f.a, j);
                        const float qb = __shfl_sync(ALL, qf, j);
                        if (b == e.a) q += qb;
                    }
                }
            }
            if (e.a >= own.x && e.a < own.y) out[e.a] = from_f<T>(grad_of<false>(e.x, r, r.l0, -w * q, R.inv_t));
        }
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
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

int sb_distill_loss(const sb_logits* x, const sb_distill* d, void* stream) {
    Rows R;
    int rc = check_rows(x, &R);
    if (rc != SB_OK || (rc = check_distill(x, d)) != SB_OK || x->n_rows == 0) return rc;
    if (!d->loss || !aligned(d->loss, 4)) return fail(SB_E_ARG, "loss is NULL or not aligned to its type");
    if (R.a <= SMALL) return small_distill(x, *d, (cudaStream_t)stream);
    return dispatch(x, wide_forward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int lists = M == SB_MASK_NONE ? 0 : WARPS * PASS_BYTES;
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
    if (!aligned(grad, x->dtype == SB_DTYPE_F32 ? 4 : 2) || !aligned(g_loss, 4))
        return fail(SB_E_ARG, "grad or g_loss not aligned to its type");
    if (R.a <= SMALL) return small_distill_backward(x, *d, g_loss, g_loss_stride, grad, (cudaStream_t)stream);
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
