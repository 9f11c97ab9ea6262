// block_write.hip -- queries and keys normed by head and turned to their positions,
// keys and values quantised with block scales into their slots, in one pass.
//
//   y = x * rsqrt(sum(x^2)/D + eps) * w,   (a, b) -> (a c - b s, a s + b c)
//   E = the smallest whole number with max|y| <= M 2^E over 32 neighbours,
//   code = y / 2^E rounded to the nearest code (M: the largest one)
//
// Rows are cut into units as in norm_rotate.hip: what a rotation pairs is in one
// lane.  A wave takes query rows or K/V rows of one token, not a mixture: queries are
// computed in 32 bits, keys in 64 (from eps and factor, which are 32-bit numbers) and
// rounded to 32 before they are quantised, so that a code does not hang on the noise of
// the sums.  64-bit arithmetic runs at the rate of
// scalar 32-bit arithmetic here and the memory hides it: 32768 tokens, written and read
// back, took 211 us with it and 209 with keys in 32 bits (measured when K and V still
// had waves of their own).  A block's 32 values lie in lanes as the rotation wants them,
// so finished rows pass through LDS (of the wave's own) and come back as 16 neighbours a
// lane, two lanes to a block.  Where a piece lies in LDS is chosen so that 16 lanes meet
// all banks (32768 tokens of 32 + 2 x 8 heads of 128, 8 bits: 165 us with rows and turns
// in order, two thirds of them with the LDS held by conflicts; 145 so).
//
// Bound by memory where tokens are many (those 145 us: 5.1 TB/s; 8192 tokens 37.3), by
// the launch and the chain of loads where they are few (16 tokens: 5.0 us).
#include "block_scale.h"
#include "norm_rotate.h"

namespace kvec {

struct BwArgs {
    NrArgs n;
    uint32_t half;                            // bytes of a half record
    uint32_t q_pieces, k_pieces;              // waves of a token's queries; of its keys (or keys and values)
    FastDiv by_pieces;
    uint32_t items;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr double kTwoPiHi = 6.283185307179586477;        // 2 pi rounded to 64 bits,
constexpr double kTwoPiLo = 2.449293598294706414e-16;    // and what that leaves out

// cos and sin of position * frequency, the product reduced to half a turn with
// 64 bits and more.
__device__ __forceinline__ void turn_of(double x, float factor, float* c, float* s) {
    const double n = __builtin_rint(x * 0.15915494309189533577);
    const double r = __builtin_fma(-n, kTwoPiLo, __builtin_fma(-n, kTwoPiHi, x));
    sincospif(float(r * 0.31830988618379067154), s, c);
    *c *= factor;
    *s *= factor;
}
__device__ __forceinline__ void turn_of(double x, float factor, double* c, double* s) {
    const double n = __builtin_rint(x * 0.15915494309189533577);
    const double r = __builtin_fma(-n, kTwoPiLo, __builtin_fma(-n, kTwoPiHi, x));
    sincospi(r * 0.31830988618379067154, s, c);
    *c *= double(factor);
    *s *= double(factor);
}

__device__ __forceinline__ float inv_root(float x) { return 1.0f / sqrtf(x); }
__device__ __forceinline__ double inv_root(double x) { return 1.0 / sqrt(x); }

template <class F>
struct Turn {
    F c, s;
};

// Where turn i lies in LDS.  Lanes read eight in a row each, 64 or 128 bytes apart; so
// that neighbours meet other banks, places within the eight go by the lane.
template <class F>
__device__ __forceinline__ uint32_t turn_at(uint32_t i) {
    return sizeof(F) == 8 ? i ^ (i >> 4 & 7) : i ^ (i >> 5 & 3) << 1;
}
// Where 16 bytes x of a staged row lie, in pieces of 16 bytes.  They are written one in
// two or four, two or more rows at once (`rows`: by the row's number), and read one in
// four: with both, 16 lanes meet all banks from rows of 256 bytes on.
struct Place {
    uint32_t rows;
    __device__ __forceinline__ Place(uint32_t group, uint32_t pieces) : rows(((group & 1) * 3 ^ (group >> 1 & 1) * 10) & (pieces - 1)) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return x ^ rows ^ (x >> 4 & 3); }
};

// Where a lane's units lie in its row.
template <int W, int NU>
struct Units {
    uint32_t a[NU], b[NU], pair[NU];
    bool turned[NU];
    __device__ __forceinline__ Units(const NrArgs& p, uint32_t sub, uint32_t lanes) {
#pragma unroll
        for (int n = 0; n < NU; ++n) unit_at<W>(p, sub + n * lanes, a[n], b[n], pair[n], turned[n]);
    }
};

// ITER rows of a group, loaded together: row0, row0 + step, ..
template <class T, int W, int NU, int ITER>
struct Rows {
    Raw<T, W> a[ITER][NU], b[ITER][NU];
    __device__ __forceinline__ void load(const NrArgs& p, const Units<W, NU>& u, const uint8_t* base, int64_t hs, uint32_t row0,
                                         uint32_t step, uint32_t rows) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const uint32_t r = row0 + i * step;
            const T* x = reinterpret_cast<const T*>(base) + int64_t(r) * hs;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                a[i][n] = Raw<T, W>{};
                b[i][n] = Raw<T, W>{};
                if (r < rows && u.a[n] < p.dim) a[i][n].load(x + u.a[n]);
                if (r < rows && u.b[n] < p.dim) b[i][n].load(x + u.b[n]);
            }
        }
    }
};

// A row normed and turned, in F; a and b: its units' chunks.
template <class F, class T, int W, int NU>
__device__ __forceinline__ void norm_turn(const NrArgs& p, const Units<W, NU>& u, uint32_t lanes, const uint8_t* weight,
                                          const Turn<F>* turn, F (*a)[W], F (*b)[W]) {
    if (p.norm) {
        F ss = 0;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int j = 0; j < W; ++j) ss += a[n][j] * a[n][j] + b[n][j] * b[n][j];
        for (uint32_t d = lanes >> 1; d; d >>= 1) ss += __shfl_xor(ss, int(d), 64);
        const F inv = inv_root(ss / F(p.dim) + F(p.eps));
        const T* w = reinterpret_cast<const T*>(weight);
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            float wa[W], wb[W];
#pragma unroll
            for (int j = 0; j < W; ++j) wa[j] = wb[j] = 1.0f;
            Raw<T, W> raw;
            if (w && u.a[n] < p.dim) {
                raw.load(w + u.a[n]);
                raw.get(wa);
            }
            if (w && u.b[n] < p.dim) {
                raw.load(w + u.b[n]);
                raw.get(wb);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                a[n][j] *= inv * F(wa[j]);
                b[n][j] *= inv * F(wb[j]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        if (!u.turned[n]) continue;
        if (W > 1 && p.interleaved) {
            // pairs of neighbours: the first W/2 in a, the rest in b
#pragma unroll
            for (int j = 0; j < W / 2; ++j) {
                const Turn<F> c0 = turn[turn_at<F>(u.pair[n] + j)], c1 = turn[turn_at<F>(u.pair[n] + W / 2 + j)];
                const F x0 = a[n][2 * j], y0 = a[n][2 * j + 1], x1 = b[n][2 * j], y1 = b[n][2 * j + 1];
                a[n][2 * j] = x0 * c0.c - y0 * c0.s;
                a[n][2 * j + 1] = x0 * c0.s + y0 * c0.c;
                b[n][2 * j] = x1 * c1.c - y1 * c1.s;
                b[n][2 * j + 1] = x1 * c1.s + y1 * c1.c;
            }
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const Turn<F> c = turn[turn_at<F>(u.pair[n] + j)];
                const F x = a[n][j], y = b[n][j];
                a[n][j] = x * c.c - y * c.s;
                b[n][j] = x * c.s + y * c.c;
            }
        }
    }
}

// The token's cos and sin, into a wave's part of LDS.
template <class F>
__device__ __forceinline__ void make_turns(const NrArgs& p, uint32_t t, uint32_t lane, Turn<F>* turn) {
    const uint32_t half = p.rot / 2;
    for (uint32_t i = lane; i < half; i += 64) {
        const uint32_t ax = p.axis_of ? min(uint32_t(p.axis_of[i]), p.axes - 1) : 0u;
        Turn<F>& to = turn[turn_at<F>(i)];
        turn_of(double(p.pos[int64_t(ax) * p.axis_stride + t]) * p.freqs[i], p.factor, &to.c, &to.s);
    }
    wave_order();
}

// A lane's units of a finished row as 32-bit values in LDS.
template <int W, int NU>
__device__ __forceinline__ void stage(const NrArgs& p, const Units<W, NU>& u, const Place& place, float* row, const float (*a)[W],
                                      const float (*b)[W]) {
    auto put = [&](uint32_t at, const float* x) __attribute__((always_inline)) {
        if (at >= p.dim) return;
        if constexpr (W == 8) {
            f32x4* to = reinterpret_cast<f32x4*>(row);
            to[place(at / 4)] = f32x4{x[0], x[1], x[2], x[3]};
            to[place(at / 4 + 1)] = f32x4{x[4], x[5], x[6], x[7]};
        } else {
            row[place(at / 4) * 4 + at % 4] = x[0];
        }
    };
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        put(u.a[n], a[n]);
        put(u.b[n], b[n]);
    }
}

// Row `r` of a half record out of LDS: 16 neighbours a lane, two lanes a block.
template <class T, int BITS>
__device__ __forceinline__ void quantise(const NrArgs& p, const Place& place, const float* row, uint8_t* half, uint32_t r, uint32_t sub,
                                         bool live) {
    const bool mine = sub * 16 < p.dim;
    float y[16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f32x4 x = {0, 0, 0, 0};
        if (mine) x = reinterpret_cast<const f32x4*>(row)[place(sub * 4 + i)];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * i + j] = x[j];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    }
    top = max(top, uint32_t(__shfl_xor(int(top), 1, 64)));
    if (!mine || !live) return;
    const uint32_t byte = scale_byte<T, BITS>(top);
    uint32_t code[4];
    codes16<T, BITS>(y, byte, code);
    uint8_t* to = half + (r * p.dim + sub * 16) * BITS / 8;
    if constexpr (BITS == 8) st16(to, u32x4{code[0], code[1], code[2], code[3]});
    else *as_global(reinterpret_cast<u32x2*>(to)) = u32x2{code[0], code[1]};
    if (!(sub & 1)) *as_global(half + p.kv_heads * p.dim * BITS / 8 + (r * p.dim + sub * 16) / kScaleBlock) = uint8_t(byte);
}

// QITER: query rows of a group that a wave takes.  Where that is more than one, a wave
// takes keys and values of the same heads, too, so that the lines of a record are written
// by one; where waves are few each takes one of the two (launch_block_write).
template <class T, int BITS, int W, int NU, int QITER>
__global__ __launch_bounds__(kNRB) void block_write_kernel(BwArgs g) {
    constexpr int WAVES = kNRB / 64;
    constexpr bool BOTH = QITER > 1;
    __shared__ __attribute__((aligned(16))) Turn<double> turns[WAVES][kMaxBlockDim / 2];
    __shared__ __attribute__((aligned(16))) float rows_of[WAVES][1024];
    const NrArgs& p = g.n;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item = blockIdx.x * WAVES + wave;
    if (item >= g.items) return;
    const uint32_t t = fdiv(item, g.by_pieces);
    uint32_t piece = item - t * g.by_pieces.d;
    if (p.n_tokens && int64_t(t) >= int64_t(*p.n_tokens)) return;
    const uint32_t lanes = 1u << p.lg, sub = lane & (lanes - 1), group = lane >> p.lg, groups = 64u >> p.lg;
    const Units<W, NU> u(p, sub, lanes);
    if (piece < g.q_pieces) {
        const uint32_t row0 = piece * (groups * QITER) + group;
        Rows<T, W, NU, QITER> x;
        x.load(p, u, p.q + int64_t(t) * p.qs * int64_t(sizeof(T)), p.qh, row0, groups, p.heads);
        Turn<float>* turn = reinterpret_cast<Turn<float>*>(turns[wave]);
        make_turns(p, t, lane, turn);
#pragma unroll
        for (int i = 0; i < QITER; ++i) {
            const uint32_t r = row0 + i * groups;
            float a[NU][W], b[NU][W];
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                x.a[i][n].get(a[n]);
                x.b[i][n].get(b[n]);
            }
            norm_turn<float, T, W, NU>(p, u, lanes, p.wq, turn, a, b);
            if (r >= p.heads) continue;
            T* y = reinterpret_cast<T*>(p.o) + int64_t(t) * p.os + int64_t(r) * p.oh;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if (u.a[n] < p.dim) put<T, W>(y + u.a[n], a[n]);
                if (u.b[n] < p.dim) put<T, W>(y + u.b[n], b[n]);
            }
        }
        return;
    }
    piece -= g.q_pieces;
    const int32_t slot = p.slots[t];
    if (slot < 0 || int64_t(slot) >= p.n_slots) return;
    bool keys = true, values = true;
    if (!BOTH) {
        keys = piece < g.k_pieces;
        values = !keys;
        if (values) piece -= g.k_pieces;
    }
    const uint32_t r = piece * groups + group;
    Rows<T, W, NU, 1> xk, xv;
    if (keys) xk.load(p, u, p.k + int64_t(t) * p.ks * int64_t(sizeof(T)), p.kh, r, 0, p.kv_heads);
    if (values) xv.load(p, u, p.v + int64_t(t) * p.vs * int64_t(sizeof(T)), p.vh, r, 0, p.kv_heads);
    // a row's place in LDS: what its lanes hold, a power of two
    const uint32_t pieces = lanes * (2 * W * NU) / 4;
    const Place place(group, pieces);
    float* row = rows_of[wave] + group * pieces * 4;
    uint8_t* half = p.pool + int64_t(slot) * 2 * int64_t(g.half);
    float a[NU][W], b[NU][W];
    if (keys) {
        Turn<double>* turn = turns[wave];
        make_turns(p, t, lane, turn);
        double c[NU][W], d[NU][W];
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            xk.a[0][n].get(a[n]);
            xk.b[0][n].get(b[n]);
#pragma unroll
            for (int j = 0; j < W; ++j) c[n][j] = double(a[n][j]), d[n][j] = double(b[n][j]);
        }
        norm_turn<double, T, W, NU>(p, u, lanes, p.wk, turn, c, d);
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int j = 0; j < W; ++j) a[n][j] = float(c[n][j]), b[n][j] = float(d[n][j]);
        stage<W, NU>(p, u, place, row, a, b);
        wave_order();
        quantise<T, BITS>(p, place, row, half, r, sub, r < p.kv_heads);
        wave_order();
    }
    if (values) {
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            xv.a[0][n].get(a[n]);
            xv.b[0][n].get(b[n]);
        }
        stage<W, NU>(p, u, place, row, a, b);
        wave_order();
        quantise<T, BITS>(p, place, row, half + g.half, r, sub, r < p.kv_heads);
    }
}

typedef void (*BwFn)(BwArgs);

template <class T, int BITS>
BwFn pick_bw(bool wide, bool deep) {
    if constexpr (!__is_same(T, float)) {
        if (deep) return &block_write_kernel<T, BITS, 8, 1, 4>;
    }
    return wide ? &block_write_kernel<T, BITS, 8, 1, 1> : &block_write_kernel<T, BITS, 1, 2, 1>;
}
template <class T>
BwFn pick_bw_bits(int bits, bool wide, bool deep) {
    return bits == 8 ? pick_bw<T, 8>(wide, deep) : pick_bw<T, 4>(wide, deep);
}

int launch_block_write(const NrArgs& n, int64_t tokens, int dtype, int pool_dtype, bool wide, const char* fn, void* stream) {
    if (!aligned16(n.pool)) return set_error(KVEC_EINVAL, "%s: pool not 16-byte aligned", fn);
    BwArgs a{};
    a.n = n;
    const uint64_t half = half_bytes(int(n.kv_heads), int(n.dim), pool_dtype);
    if (half >= kMaxBlockHalf) return set_error(KVEC_EUNSUPPORTED, "%s: token record too large", fn);
    a.half = uint32_t(half);
    const uint32_t groups = 64u >> n.lg;
    const uint32_t k_pieces = (n.kv_heads + groups - 1) / groups, q1 = (n.heads + groups - 1) / groups;
    // Measured, us, one query row a group and four with K and V together, 8 bits: 32 + 2 x 8
    // heads of 128, bf16, 512 tokens 5.9, 7.2; 2048 14.6, 13.4; 8192 40.6, 37.3; 16384 90.4,
    // 75.9; 32768 174.7, 142.2.  16 + 2 x 4 heads, 1024 tokens 5.7, 7.6; 4096 17.2, 17.5;
    // 16384 49.8, 47.6.  64 + 2 x 8, 2048 tokens 19.8, 20.6; 16384 143.7, 123.9.  Four rows
    // lose at any size where the heads are one row a group (8 + 2 x 2 of 64, 16384 tokens
    // 39.0, 42.9; 65536 140, 156) and in 32 bits, whose rows take twice the registers (32 + 2
    // x 8 of 128, 8192 tokens 63.0, 68.3; 64 + 2 x 8, 32768 423, 446).  So: 16-bit values,
    // two rows a group or more, and waves of single rows for the card twice over.
    const bool deep = wide && dtype != KVEC_F32 && q1 > 1 && uint64_t(tokens) * (q1 + 2 * k_pieces) >= 2 * 256 * 32;
    a.q_pieces = deep ? (q1 + 3) / 4 : q1;
    a.k_pieces = k_pieces;
    const uint64_t pieces = uint64_t(a.q_pieces) + (deep ? k_pieces : 2 * k_pieces), items = uint64_t(tokens) * pieces;
    if (!launchable((items + 3) / 4, kNRB)) return set_error(KVEC_EUNSUPPORTED, "%s: too many rows for one launch", fn);
    a.by_pieces = make_fastdiv(uint32_t(pieces));
    a.items = uint32_t(items);
    const int bits = block_bits(pool_dtype);
    BwFn f = dtype == KVEC_F32 ? pick_bw_bits<float>(bits, wide, deep)
             : dtype == KVEC_BF16 ? pick_bw_bits<__bf16>(bits, wide, deep)
                                  : pick_bw_bits<_Float16>(bits, wide, deep);
    hipLaunchKernelGGL(f, dim3(unsigned((items + 3) / 4)), dim3(kNRB), 0, as_stream(stream), a);
    return check_launch(fn);
}

}  // namespace kvec
