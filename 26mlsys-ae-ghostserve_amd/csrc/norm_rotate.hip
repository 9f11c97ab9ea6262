// norm_rotate.hip -- queries and keys normed by head and turned to their
// positions, keys and values written to their slots of the pool, in one pass.
//
//   y = x * rsqrt(sum(x^2)/D + eps) * w,   (a, b) -> (a c - b s, a s + b c)
//
// A head's values are one row; q, k and v rows of a token are read once and
// written once, and nothing else is large: the kernel is bound by HBM.  A row
// is cut into units of two chunks of W values that a rotation pairs (x[i..],
// x[i + rot/2..]; or 2 W neighbours when pairs are neighbours; or 2 W values
// that are not turned).  A group of 2^lg lanes holds a row, one unit a lane (W = 8:
// two 16-byte loads), the sum of squares is reduced inside the group, and one
// wave takes ITER x (64 / 2^lg) rows of one token with all their loads in
// flight before the first is used.  A wave's cos and sin are made once for its
// rows, one frequency a lane, and handed round through LDS: the angle in turns
// is a 64-bit product less its nearest integer, so far positions keep theirs,
// and only the remainder (at most half a turn) goes to 32 bits.  No wave waits
// for another, so there is no barrier.
//
// Measured: 32768 tokens of 32 + 2 x 8 heads of 128, bf16: 156 us, 5.2 TB/s (a copy
// reaches 6.0); 3998 tokens of 32 + 2 x 4 heads, fp16 into fp8, 20.4 us, 3.8 TB/s, of
// which the quotients by the scales are 0.7; 5001 tokens on three axes 20 us, 4.6
// TB/s; 16 tokens 4.4 us.  8192 tokens of 32 + 2 x 8 heads of 128: bf16 35 us, 5.7
// TB/s, float32 77 us, 5.2 TB/s, float32 into fp8 67 us, 5.3 TB/s.  Where pairs lie in
// no whole 16-byte chunks (heads of 80 half turned) or rows start off 16 bytes a lane
// takes one value at a time: 194 and 191 us, 0.65 and 1.06 TB/s.
#include "norm_rotate.h"

namespace kvec {

template <class T, class PT, int W, int NU, int ITER>
__global__ __launch_bounds__(kNRB) void norm_rotate_kernel(NrArgs p) {
    __shared__ f32x2 turn[kNRB / 64][kMaxHalf];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t item = blockIdx.x * (kNRB / 64) + wave;
    if (item >= p.items) return;
    const uint32_t t = fdiv(item, p.div_chunks), piece = item - t * p.div_chunks.d;
    if (p.n_tokens && int64_t(t) >= int64_t(*p.n_tokens)) return;
    const uint32_t lanes = 1u << p.lg, sub = lane & (lanes - 1), group = lane >> p.lg, groups = 64u >> p.lg;
    const uint32_t rows = p.heads + 2 * p.kv_heads;
    const uint32_t row0 = piece * (groups * ITER) + group;
    const int32_t slot = p.slots[t];
    const bool kept = slot >= 0 && int64_t(slot) < p.n_slots;

    uint32_t ua[NU], ub[NU], up[NU];
    bool ut[NU];
#pragma unroll
    for (int n = 0; n < NU; ++n) unit_at<W>(p, sub + n * lanes, ua[n], ub[n], up[n], ut[n]);

    // every load of the wave's rows
    Raw<T, W> xa[ITER][NU], xb[ITER][NU];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const uint32_t r = row0 + i * groups;
        const T* x;
        if (r < p.heads) x = reinterpret_cast<const T*>(p.q) + int64_t(t) * p.qs + int64_t(r) * p.qh;
        else if (r < p.heads + p.kv_heads)
            x = reinterpret_cast<const T*>(p.k) + int64_t(t) * p.ks + int64_t(r - p.heads) * p.kh;
        else x = reinterpret_cast<const T*>(p.v) + int64_t(t) * p.vs + int64_t(r - p.heads - p.kv_heads) * p.vh;
        const bool live = r < rows && (r < p.heads || kept);
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            xa[i][n] = Raw<T, W>{};
            xb[i][n] = Raw<T, W>{};
            if (live && ua[n] < p.dim) xa[i][n].load(x + ua[n]);
            if (live && ub[n] < p.dim) xb[i][n].load(x + ub[n]);
        }
    }

    // the token's angles
    const uint32_t half = p.rot / 2;
    for (uint32_t i = lane; i < half; i += 64) {
        const uint32_t ax = p.axis_of ? min(uint32_t(p.axis_of[i]), p.axes - 1) : 0u;
        const double x = double(p.pos[int64_t(ax) * p.axis_stride + t]) * p.freqs[i] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * float(x - __builtin_rint(x)), &s, &c);
        turn[wave][i] = f32x2{c * p.factor, s * p.factor};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

    const float k_scale = p.k_scale ? *p.k_scale : 1.0f, v_scale = p.v_scale ? *p.v_scale : 1.0f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const uint32_t r = row0 + i * groups;
        const bool is_q = r < p.heads, is_k = !is_q && r < p.heads + p.kv_heads;
        float a[NU][W], b[NU][W];
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            xa[i][n].get(a[n]);
            xb[i][n].get(b[n]);
        }
        if (p.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int n = 0; n < NU; ++n)
#pragma unroll
                for (int j = 0; j < W; ++j) ss += a[n][j] * a[n][j] + b[n][j] * b[n][j];
            for (uint32_t d = lanes >> 1; d; d >>= 1) ss += __shfl_xor(ss, d, 64);
            if (is_q || is_k) {
                const float inv = 1.0f / sqrtf(ss / float(p.dim) + p.eps);
                const T* w = reinterpret_cast<const T*>(is_q ? p.wq : p.wk);
#pragma unroll
                for (int n = 0; n < NU; ++n) {
                    float wa[W], wb[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) wa[j] = wb[j] = 1.0f;
                    Raw<T, W> raw;
                    if (w && ua[n] < p.dim) {
                        raw.load(w + ua[n]);
                        raw.get(wa);
                    }
                    if (w && ub[n] < p.dim) {
                        raw.load(w + ub[n]);
                        raw.get(wb);
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        a[n][j] *= inv * wa[j];
                        b[n][j] *= inv * wb[j];
                    }
                }
            }
        }
        if (is_q || is_k) {
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if (!ut[n]) continue;
                if (W > 1 && p.interleaved) {
                    // pairs of neighbours: the first W/2 in a, the rest in b
#pragma unroll
                    for (int j = 0; j < W / 2; ++j) {
                        const f32x2 c0 = turn[wave][up[n] + j], c1 = turn[wave][up[n] + W / 2 + j];
                        const float x0 = a[n][2 * j], y0 = a[n][2 * j + 1], x1 = b[n][2 * j], y1 = b[n][2 * j + 1];
                        a[n][2 * j] = x0 * c0.x - y0 * c0.y;
                        a[n][2 * j + 1] = x0 * c0.y + y0 * c0.x;
                        b[n][2 * j] = x1 * c1.x - y1 * c1.y;
                        b[n][2 * j + 1] = x1 * c1.y + y1 * c1.x;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const f32x2 c = turn[wave][up[n] + j];
                        const float x = a[n][j], y = b[n][j];
                        a[n][j] = x * c.x - y * c.y;
                        b[n][j] = x * c.y + y * c.x;
                    }
                }
            }
        }
        if (r >= rows || !(is_q || kept)) continue;
        if (is_q) {
            T* y = reinterpret_cast<T*>(p.o) + int64_t(t) * p.os + int64_t(r) * p.oh;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if (ua[n] < p.dim) put<T, W>(y + ua[n], a[n]);
                if (ub[n] < p.dim) put<T, W>(y + ub[n], b[n]);
            }
        } else {
            // record of the slot: [2][kv_heads][dim]
            PT* y = reinterpret_cast<PT*>(p.pool) +
                    (int64_t(slot) * 2 * p.kv_heads + (r - p.heads)) * int64_t(p.dim);
            if constexpr (!__is_same(T, PT)) {
                // a quotient, not a product with the reciprocal: that is off by a step
                // at midpoints, and infinite under 2^-128
                const float f = is_k ? k_scale : v_scale;
#pragma unroll
                for (int n = 0; n < NU; ++n)
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        a[n][j] /= f;
                        b[n][j] /= f;
                    }
            }
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if (ua[n] < p.dim) put<PT, W>(y + ua[n], a[n]);
                if (ub[n] < p.dim) put<PT, W>(y + ub[n], b[n]);
            }
        }
    }
}

typedef void (*NrFn)(NrArgs);

template <class T, class PT>
NrFn pick_nr(bool wide, bool deep) {
    if (wide) return deep ? &norm_rotate_kernel<T, PT, 8, 1, 3> : &norm_rotate_kernel<T, PT, 8, 1, 1>;
    return &norm_rotate_kernel<T, PT, 1, 4, 1>;
}

template <class T>
NrFn pick_nr_pool(bool fp8, bool wide, bool deep) {
    return fp8 ? pick_nr<T, Fp8>(wide, deep) : pick_nr<T, T>(wide, deep);
}

}  // namespace kvec

using namespace kvec;

extern "C" int kvec_norm_rotate_write(const kvec_norm_rotate* s, void* stream) {
    static const char* fn = "kvec_norm_rotate_write";
    if (!s) return set_error(KVEC_EINVAL, "%s: null descriptor", fn);
    if (s->tokens < 0 || s->heads < 1 || s->kv_heads < 1 || s->dim < 1 || s->n_slots < 0)
        return set_error(KVEC_EINVAL, "%s: bad sizes", fn);
    if (s->dim > kMaxDim) return set_error(KVEC_EUNSUPPORTED, "%s: dim=%d past %d", fn, s->dim, kMaxDim);
    if (s->rot < 0 || s->rot > s->dim || s->rot % 2)
        return set_error(KVEC_EINVAL, "%s: rot=%d must be even and at most dim=%d", fn, s->rot, s->dim);
    if (s->dtype != KVEC_F32 && s->dtype != KVEC_BF16 && s->dtype != KVEC_F16)
        return set_error(KVEC_EINVAL, "%s: dtype %d", fn, s->dtype);
    const bool blocks = block_bits(s->pool_dtype) != 0;
    if (s->pool_dtype != s->dtype && s->pool_dtype != KVEC_FP8_E4M3 && !blocks)
        return set_error(KVEC_EINVAL, "%s: pool_dtype %d is neither dtype, fp8 nor one with block scales", fn, s->pool_dtype);
    if (s->pool_dtype != KVEC_FP8_E4M3 && (s->k_scale || s->v_scale))
        return set_error(KVEC_EINVAL, "%s: scales are an fp8 pool's", fn);
    if (blocks && (s->dim % kScaleBlock || s->dim > kMaxBlockDim))
        return set_error(KVEC_EUNSUPPORTED, "%s: dim=%d must be a multiple of %d up to %d", fn, s->dim, kScaleBlock, kMaxBlockDim);
    if (s->rot && (s->axes < 1 || s->axes > 8 || s->axis_stride < 0 || s->axis_stride > (int64_t(1) << 40)))
        return set_error(KVEC_EINVAL, "%s: axes=%d axis_stride=%lld", fn, s->axes, (long long)s->axis_stride);
    if (s->norm && !(s->eps >= 0.0f)) return set_error(KVEC_EINVAL, "%s: eps must not be negative", fn);
    if (s->tokens == 0) return KVEC_OK;
    if (!s->q || !s->k || !s->v || !s->q_out || !s->slots || (s->n_slots && !s->pool) ||
        (s->rot && (!s->positions || !s->freqs)))
        return set_error(KVEC_EINVAL, "%s: null array", fn);
    const int64_t es = type_bytes(s->dtype);
    const int64_t str[8] = {s->q_stride, s->q_head_stride, s->k_stride, s->k_head_stride,
                            s->v_stride, s->v_head_stride, s->o_stride, s->o_head_stride};
    for (int64_t x : str)
        if (x < 0 || x > (int64_t(1) << 40)) return set_error(KVEC_EINVAL, "%s: stride %lld", fn, (long long)x);
    const bool same = s->q_out == s->q && s->o_stride == s->q_stride && s->o_head_stride == s->q_head_stride;
    if (rows_overlap(s->tokens, s->o_stride, s->heads, s->o_head_stride, s->dim))
        return set_error(KVEC_EINVAL, "%s: rows of q_out overlap", fn);
    auto span = [&](const void* p, int64_t st, int64_t hs, int64_t h, const char* name) {
        return Span{p, uint64_t((s->tokens - 1) * st + (h - 1) * hs + s->dim) * uint64_t(es), name, -1};
    };
    const uint64_t pool_bytes = uint64_t(s->n_slots) * 2 * half_bytes(s->kv_heads, s->dim, s->pool_dtype);
    const Span q = span(s->q, s->q_stride, s->q_head_stride, s->heads, "q"),
               k = span(s->k, s->k_stride, s->k_head_stride, s->kv_heads, "k"),
               v = span(s->v, s->v_stride, s->v_head_stride, s->kv_heads, "v"),
               o = span(s->q_out, s->o_stride, s->o_head_stride, s->heads, "q_out"),
               pool = {s->pool, pool_bytes, "pool", -1},
               pos = {s->positions, s->rot ? uint64_t((s->axes - 1) * s->axis_stride + s->tokens) * 4 : 0, "positions", -1},
               slots = {s->slots, uint64_t(s->tokens) * 4, "slots", -1};
    int rc;
    {
        // in place, q_out lies among q's packed k and v by design
        const Span w1[1] = {pool}, r1[5] = {q, k, v, pos, slots};
        if ((rc = check_no_alias(w1, 1, r1, 5, fn))) return rc;
        const Span w2[1] = {o}, r2[6] = {pool, pos, slots, q, k, v};
        if ((rc = check_no_alias(w2, 1, r2, same ? 3 : 6, fn))) return rc;
    }
    const int half = s->rot / 2;
    // whole 16-byte chunks everywhere, and pairs that lie in whole chunks
    bool wide = s->dim % 8 == 0 && half % 8 == 0 && aligned16(s->q) && aligned16(s->k) && aligned16(s->v) &&
                aligned16(s->q_out) && aligned16(s->q_weight) && aligned16(s->k_weight) && aligned16(s->pool);
    for (int64_t x : str) wide = wide && (x * es) % 16 == 0;
    const uint32_t W = wide ? 8 : 1;
    const uint32_t units = uint32_t(half) / W + (uint32_t(s->dim - s->rot) + 2 * W - 1) / (2 * W);
    NrArgs a{};
    while ((1u << a.lg) < units && a.lg < 6) ++a.lg;
    const uint32_t groups = 64u >> a.lg, rows = uint32_t(s->heads) + 2 * uint32_t(s->kv_heads);
    // A wave takes three rows of each group where there are waves for the card
    // twelve times over: what the rows share is loaded once.  Fewer are spread out
    // (latency, and the data lies in the caches between kernels then).  Measured,
    // us, one row and three: 32 + 2 x 8 heads of 128, 4096 tokens 20.3, 23.3; 16384
    // 82.5, 84.5; 32768 164.7, 158.3; three axes, 28 + 2 x 4 heads, 8192 tokens 29.1,
    // 31.6; 16384 69.9, 67.6; 65536 270.9, 246.7.
    const uint64_t waves1 = uint64_t(s->tokens) * ((rows + groups - 1) / groups);
    const bool deep = wide && waves1 >= 12 * 256 * 32;
    if (s->tokens >= (int64_t(1) << 32)) return set_error(KVEC_EUNSUPPORTED, "%s: too many rows for one launch", fn);
    const uint32_t per = groups * (deep ? 3 : 1), chunks = (rows + per - 1) / per;
    if (!blocks && !launchable((uint64_t(s->tokens) * chunks + 3) / 4, kNRB))
        return set_error(KVEC_EUNSUPPORTED, "%s: too many rows for one launch", fn);
    a.q = (const uint8_t*)s->q;
    a.k = (const uint8_t*)s->k;
    a.v = (const uint8_t*)s->v;
    a.o = (uint8_t*)s->q_out;
    a.qs = s->q_stride, a.qh = s->q_head_stride, a.ks = s->k_stride, a.kh = s->k_head_stride;
    a.vs = s->v_stride, a.vh = s->v_head_stride, a.os = s->o_stride, a.oh = s->o_head_stride;
    a.wq = (const uint8_t*)s->q_weight;
    a.wk = (const uint8_t*)s->k_weight;
    a.pos = s->positions;
    a.axis_stride = s->axis_stride;
    a.axis_of = s->axis_of;
    a.freqs = s->freqs;
    a.pool = (uint8_t*)s->pool;
    a.slots = s->slots;
    a.k_scale = s->k_scale;
    a.v_scale = s->v_scale;
    a.n_tokens = s->n_tokens;
    a.n_slots = s->n_slots;
    a.div_chunks = make_fastdiv(chunks);
    a.items = uint32_t(s->tokens) * chunks;
    a.heads = uint32_t(s->heads);
    a.kv_heads = uint32_t(s->kv_heads);
    a.dim = uint32_t(s->dim);
    a.rot = uint32_t(s->rot);
    a.axes = uint32_t(s->axes < 1 ? 1 : s->axes);
    a.norm = s->norm;
    a.interleaved = s->interleaved;
    a.eps = s->eps;
    a.factor = s->factor;
    if (blocks) return launch_block_write(a, s->tokens, s->dtype, s->pool_dtype, wide, fn, stream);
    const bool fp8 = s->pool_dtype == KVEC_FP8_E4M3;
    NrFn f = s->dtype == KVEC_F32 ? pick_nr_pool<float>(fp8, wide, deep)
             : s->dtype == KVEC_BF16 ? pick_nr_pool<__bf16>(fp8, wide, deep)
                                     : pick_nr_pool<_Float16>(fp8, wide, deep);
    hipLaunchKernelGGL(f, dim3((a.items + 3) / 4), dim3(kNRB), 0, as_stream(stream), a);
    return check_launch(fn);
}
