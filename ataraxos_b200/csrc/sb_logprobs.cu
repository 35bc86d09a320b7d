// sb_logprobs.cu -- log-probabilities of given actions, entropy and the likeliest
// alternatives of policy rows, and their gradient.
#include "sb_policy.cuh"

namespace sb {
namespace {

// ---- forward: given actions, entropy, top alternatives -----------------------------

// One pass over the row for (M, Z, H), the action's logit beside it, then the
// outputs.  Masked rows are bound by the chain mask -> legal actions -> their
// logits and by instructions (730 a row): 65,536 bf16 rows of 10,000 with bit
// masks 60 us (144 MB, 2.4 TB/s), 4096 with u8 masks 12.2 us (45 MB, 3.7 TB/s).
// Unmasked rows by latency and instructions: 2049 f32 rows of 9999 with top 8
// 27.8 us (82 MB, 2.9 TB/s).
template <typename T, int MASK, int W, bool TOP>
__device__ __forceinline__ void logprobs_rows(const Rows& R, const sb_logprobs& o) {
    extern __shared__ uint4 dyn[];
    __shared__ Sum sums[WARPS];
    __shared__ float top_x[WARPS][32];
    __shared__ int top_a[WARPS][32];
    __shared__ int counts[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = W == 1 ? 0 : warp, tid = W == 1 ? lane : threadIdx.x;
    uint8_t* sh = reinterpret_cast<uint8_t*>(dyn);
    const int row_bytes = MASK == SB_MASK_NONE ? 0 : bits_bytes(R.a);
    uint8_t* sh_bits = sh + (W == 1 ? warp * row_bytes : 0);
    uint16_t* list = reinterpret_cast<uint16_t*>(sh + (WARPS / W) * row_bytes + warp * PASS_BYTES);
    const float c = R.inv_t * LOG2E;
    const int64_t step = (int64_t)gridDim.x * (WARPS / W);
    for (int64_t row = (int64_t)blockIdx.x * (WARPS / W) + (W == 1 ? warp : 0); row < R.n; row += step) {
        const T* x = static_cast<const T*>(R.x) + row * R.stride;
        // the action's logit is asked for only when its mask is on the way too:
        // a warp that waits for the action issues no other load
        const int64_t act = o.actions ? load_index(o.actions, o.action_bytes, row) : -1;
        float xa = 0.f;
        Sum s = no_sum();
        Top top;
        top.init(TOP ? o.top : 1);
        bool joined = false;  // the first warp's list is the row's
        bool dense = MASK == SB_MASK_NONE;
        // the whole row, with up to `limit` candidates for its k best
        auto read_whole = [&](auto f, int limit) {
            constexpr int F = decltype(f)::kind;
            const LaneSum z = pass_all<T, W, true, F>(x, f, R.a, c, part);
            if (TOP) {
                top_x[warp][lane] = sorted_down<2>(z.m);
                if (tid == 0) counts[warp] = 0;
                if (W == 1) __syncwarp();
            }
            const Sum r = whole_all<T, W, true, F>(z, x, f, R.a, c, part, sums);  // synchronises four warps
            if (TOP) {
                int* count = &counts[W == 1 ? warp : 0];
                uint64_t* cand = reinterpret_cast<uint64_t*>(
                    MASK == SB_MASK_NONE ? sh + (W == 1 ? warp * 8 * CANDIDATES : 0) : reinterpret_cast<uint8_t*>(list));
                // -inf is never listed
                const float low = fmaxf(kth_peak<W>(top_x + (W == 1 ? warp : 0), o.top), -3.4028235e38f);
                if (z.m >= low) list_from<T, W, F>(low, x, f, R.a, part, cand, limit, count);
                if (W == 1) __syncwarp();
                else __syncthreads();
                joined = *count <= limit;
                if (!joined) top_of_part<T, W, F>(top, x, f, R.a, part);
                else if (part == 0) top_of_list(top, cand, *count);
            }
            return r;
        };
        bool legal;
        if (MASK == SB_MASK_NONE) {
            legal = act >= 0 && act < R.a;
            if (legal) xa = to_f(x[act]);
            s = read_whole(Filter<0>{}, W * CANDIDATES);
        } else {
            const Bits bits = stage<MASK, 32 * W>(sh_bits, R, row, tid);
            if (W == 1) __syncwarp();
            else __syncthreads();
            legal = act >= 0 && act < R.a && bits.test((int)act);
            if (legal) xa = to_f(x[act]);
            const int taken = pass_masked<T, W, true, TOP, false>(s, top, x, bits, bits, R.a, c, list, part);
            if constexpr (W == 1)
                if (taken < 0) s = read_whole(Filter<1>{bits, bits}, PASS_BYTES / 8);
            dense = W == 1 && taken < 0;
        }
        if (TOP && W > 1 && !joined) {
            top_x[warp][lane] = top.x;
            top_a[warp][lane] = top.a;
        }
        if (!dense) s = whole<W>(s, c, sums);
        else if (TOP && W > 1 && !joined) __syncthreads();
        const float2 st = stats_of(s);
        if (W == 1 || warp == 0) {
            if (lane == 0) {
                if (o.logprob) o.logprob[row] = act == -1 ? 0.f : legal ? (xa - st.x) * R.inv_t - st.y : NEG_INF;
                o.entropy[row] = st.y == INFINITY ? 0.f : st.y - LN2 * s.t / (s.n + s.r);
                if (o.row_stats) *reinterpret_cast<float2*>(o.row_stats + 2 * row) = st;
            }
            if (TOP) {
                if (W > 1 && !joined)
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

template <typename T, int MASK, int W, bool TOP>
__global__ void __launch_bounds__(WARPS * 32) logprobs_kernel(const __grid_constant__ Rows R,
                                                             const __grid_constant__ sb_logprobs o) {
    logprobs_rows<T, MASK, W, TOP>(R, o);
}

// Masked rows with alternatives, a warp each: held to 48 registers, for the
// they take 64 to 96 otherwise and the loads' latency wants the warps.  All but
// the 16-bit types under bit masks spill some of them (u8 masks have ten 16-byte
// loads in flight), and still gain in large batches.  Without -> with the cap, 20
// alternatives of 30 legal actions of 10,000, in us:
//   rows                64          4096          16,384
//   f32, u8         6.3 ->  7.8   18.9 -> 18.5   54.8 -> 52.9
//   f32, bits       5.6 ->  6.1   10.7 ->  9.0   38.1 -> 29.7
//   bf16 / f16, u8  6.6 ->  7.8   19.6 -> 17.8   56.9 -> 51.5
//   bf16 / f16, bits 5.6 -> 5.8    8.0 ->  8.3   29.5 -> 26.7
// Half of 10,000 legal, 16,384 rows: 204 -> 206 (bf16, bits) to 354 -> 307 (f32, u8).
template <typename T, int MASK>
__global__ void __launch_bounds__(WARPS * 32, 10) logprobs_top_kernel(const __grid_constant__ Rows R,
                                                                     const __grid_constant__ sb_logprobs o) {
    logprobs_rows<T, MASK, 1, true>(R, o);
}

// The gradient's bytes bound it: 65,536 bf16 rows with bit masks 266 us
// (1.46 GB, 5.5 TB/s; the zeros alone, without reading a mask, took 222 us).
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
            const int64_t a = f.top_action[row * f.top + lane];
            if (a >= 0 && a < R.a) {
                mine = (int)a;
                add = g.g_top[row * f.top + lane];
            }
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
            bits = stage<MASK, 32 * W>(sh_bits, R, row, W == 1 ? lane : threadIdx.x);
            if (W == 1) __syncwarp();
            else __syncthreads();
        }
        bool legal = act >= 0 && act < R.a;
        if (MASK != SB_MASK_NONE) legal = legal && bits.test((int)act);
        const float xm = mine >= 0 ? to_f(x[mine]) : 0.f, xa = legal ? to_f(x[act]) : 0.f;
        const float total = warp_sum(add) + (legal ? ga : 0.f);
        const RowGrad r = {st.x, st.y, -(total + gh * h), -gh, -(total + gh * h)};
        const int2 own = grad_row<T, MASK, W, true>(x, out, bits, R.a, r, R.inv_t, work, W == 1 ? 0 : warp);
        const bool same = legal && mine == (int)act;
        if (same) add += ga;
        if (mine >= own.x && mine < own.y) out[mine] = from_f<T>(grad_of<true>(xm, r, r.l0, add, R.inv_t));
        if (!__any_sync(ALL, same) && lane == 0 && legal && act >= own.x && act < own.y)
            out[act] = from_f<T>(grad_of<true>(xa, r, r.l0, ga, R.inv_t));
        if (W > 1) __syncthreads();
        else __syncwarp();
    }
}

int check_logprobs(const sb_logits* x, const sb_logprobs* o) {
    if (!o) return fail(SB_E_ARG, "outputs description is NULL");
    if (o->top < 0 || o->top > SB_POLICY_MAX_TOP) return fail(SB_E_ARG, "top must be 0..%d", SB_POLICY_MAX_TOP);
    if (o->actions && !index_bytes_ok(o->action_bytes)) return fail(SB_E_ARG, "actions must be 2, 4 or 8 bytes wide");
    if (o->actions && !aligned(o->actions, o->action_bytes)) return fail(SB_E_ARG, "actions not aligned to their type");
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
    if (!aligned(out->entropy, 4) || !aligned(out->logprob, 4) || !aligned(out->row_stats, 8) ||
        (out->top && (!aligned(out->top_action, 8) || !aligned(out->top_logprob, 4))))
        return fail(SB_E_ARG, "an output is not aligned to its type (row_stats: 8 bytes)");
    if (R.a <= SMALL) return small_logprobs(x, *out, (cudaStream_t)stream);
    return dispatch(x, wide_forward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int smem = M != SB_MASK_NONE ? WARPS / W * bits_bytes(R.a) + WARPS * PASS_BYTES
                         : out->top        ? WARPS * 8 * CANDIDATES
                                           : 0;
        const auto st = (cudaStream_t)stream;
        const unsigned grid = grid_of(R.n, W);
        if (!out->top) logprobs_kernel<T, M, W, false><<<grid, WARPS * 32, smem, st>>>(R, *out);
        else if constexpr (M != SB_MASK_NONE && W == 1) logprobs_top_kernel<T, M><<<grid, WARPS * 32, smem, st>>>(R, *out);
        else logprobs_kernel<T, M, W, true><<<grid, WARPS * 32, smem, st>>>(R, *out);
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
    if (!aligned(fwd->row_stats, 8) || !aligned(fwd->entropy, 4) || !aligned(g->g_logprob, 4) ||
        !aligned(g->g_entropy, 4) || (g->g_top && (!aligned(g->g_top, 4) || !aligned(fwd->top_action, 8))))
        return fail(SB_E_ARG, "an operand is not aligned to its type (row_stats: 8 bytes)");
    if ((g->g_logprob && !fwd->actions) || (g->g_top && (!fwd->top || !fwd->top_action)))
        return fail(SB_E_ARG, "a gradient of an output that the forward call did not have");
    if (R.a <= SMALL) return small_logprobs_backward(x, *fwd, *g, (cudaStream_t)stream);
    return dispatch(x, wide_backward(x), [&](auto* t, auto mask, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int M = decltype(mask)::value, W = decltype(w)::value;
        const int smem = M == SB_MASK_NONE ? 0 : WARPS / W * bits_bytes(R.a) + WARPS * GRAD_BYTES;
        logprobs_backward_kernel<T, M, W><<<grid_of(R.n, W), WARPS * 32, smem, (cudaStream_t)stream>>>(R, *fwd, *g);
        return launched("logprobs_backward_kernel launch");
    });
}

}  // extern "C"
