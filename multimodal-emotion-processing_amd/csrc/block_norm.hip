// mep_block_norm_fwd / _bwd: the norms around a block, fused with its gate and the residual scale:
//   stream = scale * x + gate * N(y),   normed = N'(stream)
// N(y) = yh w + b with yh = (y - mean) r (layer), y r (rms) or y (none), r = rsqrt(mean square + eps); N' likewise.
// Without x and the second norm it is the norm before a block (or of each head's row).
//
// Backward, with u = g w the gradient at the normalised row xh of a norm: dx = r (u - xh mean(u xh) - [layer] mean(u)).
//   dS = dstream + N'^T(dnormed);  dx = scale dS;  dscale = sum dS x;  dgate = sum dS N(y);  dy = N^T(gate dS)
// The stream is formed again from y and x in 32 bits (the stored one is rounded to 16), so parameter gradients kept
// in 32 bits are sums of exact terms; the four row statistics come from the forward.
//
// Bound by memory: every row is read and written once, held in registers in between: 8 elements in each of L lanes, L = 16
// of a wave to 1024 of a workgroup by the row's width, in 16-byte accesses at any address (TAIL: widths that end inside one).
// A workgroup walks many rows with the parameters, and in the backward the column sums, in registers; the sums of its row
// slots are joined in LDS, those of the workgroups by a second kernel, in a fixed order.  With 8
// elements a lane the backward (parameters, up to 5 sums and 4 rows) holds everything in about 200 registers, two waves on a SIMD: at
// 16384 rows of 4096 in bf16, both norms and a gate, 196 us (4.1 TB/s), 455 with 16 elements; the forward 119 us (4.5 TB/s).
// Rows of more than 4096 channels have 1024 lanes of 128 registers each, which does not hold the backward: it spills 93 to 441 of them, and
// 8192 rows of 8192 take 531 us (1.5 TB/s; forward 125 us, 4.3).
#include "elem.h"

namespace {

using namespace mep;

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_SEQUENCE = 2, GATE_FULL = 3 };
enum { KIND_NONE = 0, KIND_RMS = 1, KIND_LAYER = 2 };

template <int L> constexpr int norm_threads() { return L < 256 ? 256 : L; }

// sums of a and b over the L lanes of a row, in a fixed order, in every lane.  L = 16: a DPP row; 64: a wave;
// more: L / 64 waves of the workgroup, through one of red's two halves (`par`, alternated from call to call: a half is written again
// only behind the barrier of the call between, which every wave reaches after it has read the half)
template <int L>
MEP_DEV void row_sum2(float& a, float& b, float* red, int par) {
    if constexpr (L == 16) {
        a += dpp_mov<0xB1>(a); b += dpp_mov<0xB1>(b);
        a += dpp_mov<0x4E>(a); b += dpp_mov<0x4E>(b);
        a += dpp_mov<0x141>(a); b += dpp_mov<0x141>(b);
        a += dpp_mov<0x140>(a); b += dpp_mov<0x140>(b);
    } else {
        a = wave_sum(a);
        b = wave_sum(b);
        if constexpr (L > 64) {
            constexpr int W = L / 64, ALL = norm_threads<L>() / 64;
            float* r = red + par * 2 * ALL;
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) { r[2 * wave] = a; r[2 * wave + 1] = b; }
            __syncthreads();
            r += wave / W * 2 * W;
            a = r[0]; b = r[1];
#pragma unroll
            for (int i = 1; i < W; ++i) { a += r[2 * i]; b += r[2 * i + 1]; }
        }
    }
}

constexpr int E = 8;      // elements of a lane: chunk c of V covers columns (c L + lane) V ..; zeros past D

template <class T, int V, int L, bool TAIL>
MEP_DEV void load_row(const MEP_G T* p, int lane, int D, float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
        const int col = (c * L + lane) * V;
        float w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 0.f;
        if (col + V <= D) {
            load_f32<T, V>(p + col, w);
        } else if (TAIL) {
#pragma unroll
            for (int j = 0; j < V; ++j) if (col + j < D) w[j] = (float)p[col + j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) v[c * V + j] = w[j];
    }
}
template <class T, int V, int L, bool TAIL>
MEP_DEV void store_row(MEP_G T* p, int lane, int D, const float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
        const int col = (c * L + lane) * V;
        float w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = v[c * V + j];
        if (col + V <= D) {
            store_f32<T, V>(p + col, w);
        } else if (TAIL) {
#pragma unroll
            for (int j = 0; j < V; ++j) if (col + j < D) p[col + j] = (T)w[j];
        }
    }
}
// A row's elements as they lie in memory, on their way to registers a row ahead of their use
template <class T, int V> struct RawRow { typename VecOf<T, V>::type v[E / V]; };
template <class T, int V, int L, bool TAIL>
MEP_DEV void fetch_row(const MEP_G T* p, int lane, int D, RawRow<T, V>& r) {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
        const int col = (c * L + lane) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[c][j] = (T)0.f;
        if (col + V <= D) {
            r.v[c] = *reinterpret_cast<const MEP_G typename VecOf<T, V>::loose*>(p + col);
        } else if (TAIL) {
#pragma unroll
            for (int j = 0; j < V; ++j) if (col + j < D) r.v[c][j] = p[col + j];
        }
    }
}
template <class T, int V>
MEP_DEV void widen(const RawRow<T, V>& r, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)r.v[i / V][i % V];
}
// a parameter row, fp32 or the activations' type; `miss` where there is none
template <class T, int V, int L, bool TAIL>
MEP_DEV void load_param(uint64_t p, int64_t off, bool wide, float miss, int lane, int D, float (&v)[E]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = miss;
    } else if (wide) {
        load_row<float, V, L, TAIL>(G<const float>(p) + off, lane, D, v);
    } else {
        load_row<T, V, L, TAIL>(G<const T>(p) + off, lane, D, v);
    }
}


MEP_DEV float residual_scale(const mep_block_norm_desc& d) { return d.scale ? *G<const float>(d.scale) : d.scale_value; }

template <int TYPE, int V, int L, bool TAIL>
__global__ __launch_bounds__(norm_threads<L>()) void k_block_norm_fwd(mep_block_norm_desc d) {
    typedef typename ElemOf<TYPE>::T T;
    constexpr int RPB = norm_threads<L>() / L;
    __shared__ float red[L > 64 ? norm_threads<L>() / 16 : 1];
    const int lane = threadIdx.x % L, slot = threadIdx.x / L;
    const int D = d.D;
    const bool wide = d.wtype == MEP_F32, gwide = d.gtype == MEP_F32;
    const float inv = 1.0f / (float)D;
    float w[E], bi[E], nw[E], nb[E], gc[E];
    load_param<T, V, L, TAIL>(d.w, 0, wide, 1.f, lane, D, w);
    load_param<T, V, L, TAIL>(d.b, 0, wide, 0.f, lane, D, bi);
    load_param<T, V, L, TAIL>(d.nw, 0, wide, 1.f, lane, D, nw);
    load_param<T, V, L, TAIL>(d.nb, 0, wide, 0.f, lane, D, nb);
    if (d.gate_form <= GATE_CHANNEL) load_param<T, V, L, TAIL>(d.gate, 0, gwide, 1.f, lane, D, gc);
    const float sc = residual_scale(d);
    bool in[E];
#pragma unroll
    for (int i = 0; i < E; ++i) in[i] = ((i / V) * L + lane) * V + i % V < D;
    int par = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < d.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = r0 + slot;
        const bool live = row < d.rows;              // a slot past the end reduces zeros and stores nothing
        const int64_t rr = live ? row : d.rows - 1;
        float y[E], x[E];
        load_row<T, V, L, TAIL>(G<const T>(d.y) + rr * d.y_ld, lane, D, y);
        if (d.x) load_row<T, V, L, TAIL>(G<const T>(d.x) + rr * d.x_ld, lane, D, x);
        if (d.gate_form == GATE_SEQUENCE) load_param<T, V, L, TAIL>(d.gate, rr / d.T * D, gwide, 1.f, lane, D, gc);
        if (d.gate_form == GATE_FULL) load_row<T, V, L, TAIL>(G<const T>(d.gate) + rr * d.g_ld, lane, D, gc);
        float mean = 0.f, r = 1.f, smean = 0.f, sr = 1.f;
        auto stats = [&](const float (&v)[E], int kind, float& mu, float& rs) {
            if (kind == KIND_NONE) return;
            float s = 0.f, q = 0.f;
            if (kind == KIND_LAYER) {                // the mean first, then the squares around it
#pragma unroll
                for (int i = 0; i < E; ++i) s += v[i];
                row_sum2<L>(s, q, red, par);
                par ^= 1;
                mu = s * inv;
            }
            s = q = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float c = in[i] ? v[i] - mu : 0.f;
                q = fmaf(c, c, q);
            }
            row_sum2<L>(s, q, red, par);
            par ^= 1;
            rs = __frsqrt_rn(fmaf(q, inv, d.eps));
        };
        stats(y, d.kind, mean, r);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float n = fmaf((y[i] - mean) * r, w[i], bi[i]) * gc[i];
            if (d.x) n = fmaf(sc, x[i], n);
            y[i] = in[i] ? n : 0.f;
        }
        if (live) store_row<T, V, L, TAIL>(G<T>(d.stream) + row * D, lane, D, y);
        if (d.normed) {
            stats(y, d.next_kind, smean, sr);
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = fmaf((y[i] - smean) * sr, nw[i], nb[i]);
            if (live) store_row<T, V, L, TAIL>(G<T>(d.normed) + row * D, lane, D, y);
        }
        if (d.stats && live && lane == 0)
            *reinterpret_cast<MEP_G f32x4*>(G<float>(d.stats) + 4 * row) = f32x4{mean, r, smean, sr};
    }
}

// Column sums of a workgroup: partial[blockIdx.y * gridDim.x + blockIdx.x][n_sums][D] = those wanted of dw, db, dnw, dnb, dgate, and
// the scalar dscale behind all of them.  Under a sequence gate blockIdx.y is a sequence of d.T rows.  MANY: there are more sequences
// than gridDim.y, and a workgroup takes every gridDim.y-th whole one and writes its gate's gradient itself, so that the partial sums do
// not grow with the sequences (4096 of one row, 4096 channels in bf16: 8 MB and 60 us, 134 MB and 692 us with a sequence each).
template <int TYPE, int V, int L, bool TAIL, bool BIAS, bool MANY>
__global__ __launch_bounds__(norm_threads<L>(), L > 512 ? 4 : 2) void k_block_norm_bwd(mep_block_norm_bwd_desc bd) {
    typedef typename ElemOf<TYPE>::T T;
    constexpr int RPB = norm_threads<L>() / L;
    const mep_block_norm_desc& d = bd.f;
    __shared__ float red[L > 64 ? norm_threads<L>() / 16 : 1];
    __shared__ float slots[RPB > 1 ? RPB * L * E : 1];      // a column sum of each row slot
    const int lane = threadIdx.x % L, slot = threadIdx.x / L;
    const int D = d.D;
    const bool wide = d.wtype == MEP_F32, gwide = d.gtype == MEP_F32, layer = d.kind == KIND_LAYER, nlayer = d.next_kind == KIND_LAYER;
    const float inv = 1.0f / (float)D;
    const bool next = bd.dnormed != 0;
    float w[E], bi[E], nw[E], gc[E];
    load_param<T, V, L, TAIL>(d.w, 0, wide, 1.f, lane, D, w);
    load_param<T, V, L, TAIL>(BIAS ? d.b : 0, 0, wide, 0.f, lane, D, bi);
    load_param<T, V, L, TAIL>(d.nw, 0, wide, 1.f, lane, D, nw);
    if (d.gate_form <= GATE_CHANNEL) load_param<T, V, L, TAIL>(d.gate, 0, gwide, 1.f, lane, D, gc);
    else if (!MANY && d.gate_form == GATE_SEQUENCE) load_param<T, V, L, TAIL>(d.gate, (int64_t)blockIdx.y * D, gwide, 1.f, lane, D, gc);
    const float sc = residual_scale(d);
    float aw[E], ab[E], anw[E], anb[E], ag[E], as = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) aw[i] = ab[i] = anw[i] = anb[i] = ag[i] = 0.f;
    const bool by_seq = MANY || d.gate_form == GATE_SEQUENCE;
    const int nseq = MANY ? (int)(d.rows / d.T) : 0;
    int64_t first = by_seq ? (int64_t)blockIdx.y * d.T : 0, end = by_seq ? first + d.T : d.rows;
    int par = 0;
    const int64_t step = (int64_t)gridDim.x * RPB;
    RawRow<T, V> ry, rx, rg, rs, rn;
    f32x4 rst;
    auto fetch = [&](int64_t r0) {
        const int64_t rr = min(r0 + slot, end - 1);
        fetch_row<T, V, L, TAIL>(G<const T>(d.y) + rr * d.y_ld, lane, D, ry);
        if (d.x) fetch_row<T, V, L, TAIL>(G<const T>(d.x) + rr * d.x_ld, lane, D, rx);
        if (d.gate_form == GATE_FULL) fetch_row<T, V, L, TAIL>(G<const T>(d.gate) + rr * d.g_ld, lane, D, rg);
        if (bd.dstream) fetch_row<T, V, L, TAIL>(G<const T>(bd.dstream) + rr * bd.ds_ld, lane, D, rs);
        if (next) fetch_row<T, V, L, TAIL>(G<const T>(bd.dnormed) + rr * bd.dn_ld, lane, D, rn);
        rst = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(d.stats) + 4 * rr);
    };
    // v's sums over the workgroup's row slots, in order, to to(column, sum)
    auto join_slots = [&](const float (&v)[E], auto to) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) slots[slot * L * E + ((i / V) * L + lane) * V + i % V] = v[i];
        __syncthreads();
        for (int col = threadIdx.x; col < D; col += norm_threads<L>()) {
            float s = slots[col];
#pragma unroll
            for (int r = 1; r < RPB; ++r) s += slots[r * L * E + col];
            to(col, s);
        }
    };
    constexpr bool AHEAD = L < 1024;                 // 1024 threads have 128 registers each: no room for a row ahead
    for (int seq = blockIdx.y; !MANY || seq < nseq; seq += gridDim.y) {
    if constexpr (MANY) {
        load_param<T, V, L, TAIL>(d.gate, (int64_t)seq * D, gwide, 1.f, lane, D, gc);
        first = (int64_t)seq * d.T;
        end = first + d.T;
    }
    const int64_t r00 = first + (int64_t)blockIdx.x * RPB;
    if (AHEAD && r00 < end) fetch(r00);
    for (int64_t r0 = r00; r0 < end; r0 += step) {
        const int64_t row = r0 + slot;
        const bool live = row < end;                 // a slot past the end works on zeros and stores nothing
        float y[E], x[E], g[E], h[E];
        if (!AHEAD) fetch(r0);
        widen(ry, y);
        if (d.x) widen(rx, x);
        if (d.gate_form == GATE_FULL) widen(rg, gc);
        if (bd.dstream) widen(rs, g);
        if (next) widen(rn, h);
        const f32x4 st = rst;
        if (AHEAD && r0 + step < end) fetch(r0 + step);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            y[i] = (y[i] - st[0]) * st[1];           // yh
            if (!bd.dstream || !live) g[i] = 0.f;
            if (!d.x || !live) x[i] = 0.f;
        }
        if (next) {
            float su = 0.f, sq = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float n = fmaf(y[i], w[i], bi[i]) * gc[i];
                const float s = ((d.x ? fmaf(sc, x[i], n) : n) - st[2]) * st[3];   // the normalised stream
                const float hi = live ? h[i] : 0.f;  // columns past D hold zeros
                anw[i] = fmaf(hi, s, anw[i]);
                if constexpr (BIAS) anb[i] += hi;
                const float u = hi * nw[i];
                su += u;
                sq = fmaf(u, s, sq);
                h[i] = u;
            }
            if (d.next_kind != KIND_NONE) { row_sum2<L>(su, sq, red, par); par ^= 1; }
            const float mu = nlayer ? su * inv : 0.f, mq = d.next_kind != KIND_NONE ? sq * inv : 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float n = fmaf(y[i], w[i], bi[i]) * gc[i];
                const float s = ((d.x ? fmaf(sc, x[i], n) : n) - st[2]) * st[3];
                // columns past D hold values here, which meet only zeros in the sums above; they are cleared so that
                // they add nothing below
                g[i] = ((i / V) * L + lane) * V + i % V < D && live ? g[i] + st[3] * (h[i] - mu - s * mq) : 0.f;
            }
        }
        float su = 0.f, sq = 0.f, dg[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            as = fmaf(g[i], x[i], as);
            dg[i] = g[i] * fmaf(y[i], w[i], bi[i]);
            ag[i] += dg[i];
            const float dn = g[i] * gc[i];
            aw[i] = fmaf(dn, y[i], aw[i]);
            if constexpr (BIAS) ab[i] += dn;
            const float u = dn * w[i];
            x[i] = sc * g[i];
            g[i] = u;
            su += u;
            sq = fmaf(u, y[i], sq);
        }
        if (bd.dx && live) store_row<T, V, L, TAIL>(G<T>(bd.dx) + row * D, lane, D, x);
        if (bd.dgate_rows && live) store_row<T, V, L, TAIL>(G<T>(bd.dgate_rows) + row * D, lane, D, dg);
        if (d.kind != KIND_NONE) { row_sum2<L>(su, sq, red, par); par ^= 1; }
        const float mu = layer ? su * inv : 0.f, mq = d.kind != KIND_NONE ? sq * inv : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = st[1] * (g[i] - mu - y[i] * mq);
        if (live) store_row<T, V, L, TAIL>(G<T>(bd.dy) + row * D, lane, D, g);
    }
    if constexpr (!MANY) break;
    if (bd.dgate) {      // (gridDim.x is 1)
        const int64_t at = (int64_t)seq * D;
        if constexpr (RPB == 1) {
            if (gwide) store_row<float, V, L, TAIL>(G<float>(bd.dgate) + at, lane, D, ag);
            else store_row<T, V, L, TAIL>(G<T>(bd.dgate) + at, lane, D, ag);
        } else {
            join_slots(ag, [&](int col, float s) {
                if (gwide) G<float>(bd.dgate)[at + col] = s;
                else G<T>(bd.dgate)[at + col] = (T)s;
            });
        }
#pragma unroll
        for (int i = 0; i < E; ++i) ag[i] = 0.f;
    }
    }
    if (!bd.partial) return;
    const int64_t p = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    gfloat* out = G<float>(bd.partial) + p * bd.n_sums * D;
    int k = 0;
    auto put = [&](bool on, const float (&v)[E]) {
        if (!on) return;
        gfloat* o = out + (int64_t)k++ * D;
        if constexpr (RPB == 1) store_row<float, V, L, TAIL>(o, lane, D, v);
        else join_slots(v, [&](int col, float s) { o[col] = s; });
    };
    put(bd.dw != 0, aw);
    put(bd.db != 0, ab);
    put(bd.dnw != 0, anw);
    put(bd.dnb != 0, anb);
    put(bd.dgate != 0 && !MANY, ag);
    if (bd.dscale) {
        float z = 0.f;
        row_sum2<L>(as, z, red, par);
        if constexpr (RPB > 1) {
            __syncthreads();
            if (lane == 0) slots[slot] = as;
            __syncthreads();
            as = slots[0];
#pragma unroll
            for (int r = 1; r < RPB; ++r) as += slots[r];
        }
        if (threadIdx.x == 0) G<float>(bd.partial)[(int64_t)gridDim.x * gridDim.y * bd.n_sums * D + p] = as;
    }
}

// out[k][col] = sum over the partial rows, in order: 16 slices of rows per 16 columns, then the slices.
// blockIdx.y = sum * nseq + sequence for a sequence gate's sums (each sequence its own rows), else the sum.
constexpr int NORM_SUM_COLS = 16, NORM_SUM_SLICES = 16;

__global__ __launch_bounds__(NORM_SUM_COLS * NORM_SUM_SLICES) void k_block_norm_sums(mep_block_norm_bwd_desc bd, int rows_seq, int nseq) {
    const mep_block_norm_desc& d = bd.f;
    __shared__ float part[NORM_SUM_SLICES][NORM_SUM_COLS];
    const int D = d.D, c = threadIdx.x % NORM_SUM_COLS, sl = threadIdx.x / NORM_SUM_COLS;
    const uint64_t outs[5] = {bd.dw, bd.db, bd.dnw, bd.dnb, bd.dgate};
    const int all = rows_seq * nseq;
    const bool scalar = (int)blockIdx.y == (int)gridDim.y - 1 && bd.dscale;
    // which sum, and its partial rows
    int kind = 0, k = (int)blockIdx.y, seq = 0, r0 = 0, r1 = all;
    const gfloat* src;
    int64_t ld = (int64_t)bd.n_sums * D, off = 0;
    uint64_t out = 0;
    int cols = D;
    if (scalar) {
        if (blockIdx.x) return;
        src = G<const float>(bd.partial) + (int64_t)all * bd.n_sums * D;
        float s = 0.f;
        for (int i = threadIdx.x; i < all; i += NORM_SUM_COLS * NORM_SUM_SLICES) s += src[i];
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) part[0][threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) *G<float>(bd.dscale) = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
        return;
    }
    for (int i = 0, n = 0; i < 5; ++i) {
        if (!outs[i]) continue;
        const int span = i == 4 && d.gate_form == GATE_SEQUENCE ? nseq : 1;
        if (k < span) {
            kind = i;
            seq = span > 1 ? k : 0;
            if (i == 4 && d.gate_form == GATE_SEQUENCE) { r0 = k * rows_seq; r1 = r0 + rows_seq; }
            off = (int64_t)n * D;
            out = outs[i];
            break;
        }
        k -= span;
        ++n;
    }
    if (!out) return;
    src = G<const float>(bd.partial) + off;
    const int col = blockIdx.x * NORM_SUM_COLS + c;
    float s = 0.f;
    if (col < cols) {
        const int n = r1 - r0, per = (n + NORM_SUM_SLICES - 1) / NORM_SUM_SLICES;
        const int a = r0 + sl * per, b = min(r1, a + per);
#pragma unroll 8
        for (int r = a; r < b; ++r) s += src[(int64_t)r * ld + col];
    }
    part[sl][c] = s;
    __syncthreads();
    if (sl == 0 && col < cols) {
        s = part[0][c];
#pragma unroll
        for (int i = 1; i < NORM_SUM_SLICES; ++i) s += part[i][c];
        const int64_t o = (int64_t)seq * D + col;
        const int type = kind == 4 ? d.gtype : d.wtype;
        if (type == MEP_F32) G<float>(out)[o] = s;
        else if (type == MEP_BF16) G<__bf16>(out)[o] = (__bf16)s;
        else G<_Float16>(out)[o] = (_Float16)s;
    }
}

int lanes_of(int D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }
int rows_per_block(int D) {
    const int L = lanes_of(D);
    return (L < 256 ? 256 : L) / L;
}

// workgroups per sequence of the backward: as many as the compute units hold over all sequences, at least 4 rows a slot
// where there are so many (each workgroup's column sums cost 5 D floats), never more than its rows ask for; and how many
// sequences are taken side by side
dim3 bwd_grid(const mep_block_norm_desc& d, int rpb) {
    const int64_t nseq = d.gate_form == GATE_SEQUENCE ? d.rows / d.T : 1;
    const int64_t rows = d.rows / nseq;
    const int all = rpb == 1 && d.D > 2048 ? 256 : 512;      // of 512 threads and more, one fits a compute unit
    int64_t most = (all + nseq - 1) / nseq, want = (rows + 4 * rpb - 1) / (4 * rpb);
    const int64_t n = want < most ? want : most;
    return dim3((unsigned)(n < 1 ? 1 : n), (unsigned)(nseq < all ? nseq : all));
}

bool many_sequences(const mep_block_norm_desc& d, const dim3& grid) { return d.gate_form == GATE_SEQUENCE && d.rows / d.T > grid.y; }

template <int TYPE, int V, int L, bool TAIL>
void run_norm(const mep_block_norm_desc& d, const mep_block_norm_bwd_desc* b, hipStream_t st) {
    constexpr int TH = norm_threads<L>(), RPB = TH / L;
    if (!b) {
        const int64_t want = (d.rows + RPB - 1) / RPB, most = 2048;
        hipLaunchKernelGGL((k_block_norm_fwd<TYPE, V, L, TAIL>), dim3((unsigned)(want < most ? want : most)), dim3(TH), 0, st, d);
    } else {
        const dim3 grid = bwd_grid(d, RPB);
        if (many_sequences(d, grid)) hipLaunchKernelGGL((k_block_norm_bwd<TYPE, V, L, true, true, true>), grid, dim3(TH), 0, st, *b);
        else if (d.b || d.nb) hipLaunchKernelGGL((k_block_norm_bwd<TYPE, V, L, TAIL, true, false>), grid, dim3(TH), 0, st, *b);
        else hipLaunchKernelGGL((k_block_norm_bwd<TYPE, V, L, TAIL, false, false>), grid, dim3(TH), 0, st, *b);
    }
}

template <int TYPE, bool TAIL>
void pick_lanes(const mep_block_norm_desc& d, const mep_block_norm_bwd_desc* b, hipStream_t st) {
    constexpr int V = TYPE == MEP_F32 ? 4 : 8;
    switch (lanes_of(d.D)) {
        case 16: return run_norm<TYPE, V, 16, TAIL>(d, b, st);
        case 64: return run_norm<TYPE, V, 64, TAIL>(d, b, st);
        case 128: return run_norm<TYPE, V, 128, TAIL>(d, b, st);
        case 256: return run_norm<TYPE, V, 256, TAIL>(d, b, st);
        case 512: return run_norm<TYPE, V, 512, TAIL>(d, b, st);
        default: return run_norm<TYPE, V, 1024, TAIL>(d, b, st);
    }
}

template <int TYPE>
void pick_tail(const mep_block_norm_desc& d, const mep_block_norm_bwd_desc* b, hipStream_t st) {
    if (d.D % (TYPE == MEP_F32 ? 4 : 8)) pick_lanes<TYPE, true>(d, b, st);
    else pick_lanes<TYPE, false>(d, b, st);
}

void run_type(const mep_block_norm_desc& d, const mep_block_norm_bwd_desc* b, hipStream_t st) {
    if (d.type == MEP_F32) pick_tail<MEP_F32>(d, b, st);
    else if (d.type == MEP_BF16) pick_tail<MEP_BF16>(d, b, st);
    else pick_tail<MEP_F16>(d, b, st);
}

bool norm_ok(const mep_block_norm_desc& d) {
    if (d.rows < 0 || d.D < 1 || d.D > MEP_BLOCK_NORM_MAX_D || !d.y || !d.stream) return false;
    if (d.type < MEP_F32 || d.type > MEP_F16 || (d.wtype != MEP_F32 && d.wtype != d.type) ||
        (d.gtype != MEP_F32 && d.gtype != d.type)) return false;
    if (d.kind < KIND_NONE || d.kind > KIND_LAYER || d.next_kind < KIND_NONE || d.next_kind > KIND_LAYER) return false;
    if (d.gate_form == GATE_FULL && d.gtype != d.type) return false;
    if (d.gate_form < GATE_NONE || d.gate_form > GATE_FULL || (d.gate_form != GATE_NONE) != (d.gate != 0)) return false;
    if (d.gate_form == GATE_SEQUENCE && (d.T < 1 || d.rows % d.T || d.rows / d.T > 65000)) return false;
    return d.eps >= 0.f;
}

}  // namespace

extern "C" int mep_block_norm_fwd(const mep_block_norm_desc* desc, mep_stream_t stream) {
    if (!desc || !norm_ok(*desc)) { mep_set_error("mep_block_norm_fwd: invalid descriptor"); return MEP_EINVAL; }
    if (desc->rows == 0) return 0;
    run_type(*desc, nullptr, (hipStream_t)stream);
    return mep_check_launch("mep_block_norm_fwd");
}

extern "C" int mep_block_norm_partial(const mep_block_norm_desc* desc) {
    if (!desc || !norm_ok(*desc)) { mep_set_error("mep_block_norm_partial: invalid descriptor"); return MEP_EINVAL; }
    if (desc->rows == 0) return 0;
    const dim3 grid = bwd_grid(*desc, rows_per_block(desc->D));
    return (int)(grid.x * grid.y);
}

extern "C" int mep_block_norm_bwd(const mep_block_norm_bwd_desc* desc, mep_stream_t stream) {
    if (!desc || !norm_ok(desc->f) || !desc->f.stats || !desc->dy || (desc->dnormed && !desc->f.normed)) {
        mep_set_error("mep_block_norm_bwd: invalid descriptor");
        return MEP_EINVAL;
    }
    const mep_block_norm_bwd_desc& b = *desc;
    const int sums = !!b.dw + !!b.db + !!b.dnw + !!b.dnb + !!b.dgate;
    if (sums != b.n_sums || ((sums || b.dscale) && !b.partial) ||
        (b.f.gate_form == GATE_FULL ? b.dgate != 0 : b.dgate_rows != 0)) {
        mep_set_error("mep_block_norm_bwd: sums without a workspace, or a gate gradient of another form");
        return MEP_EINVAL;
    }
    if (b.f.rows == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    run_type(b.f, &b, st);
    int rc = mep_check_launch("mep_block_norm_bwd");
    if (rc || !b.partial) return rc;
    const dim3 grid = bwd_grid(b.f, rows_per_block(b.f.D));
    mep_block_norm_bwd_desc s = b;
    if (many_sequences(b.f, grid)) s.dgate = 0;      // written already
    const int ny = sums - !!b.dgate + (s.dgate ? (int)grid.y : 0) + !!b.dscale;
    if (ny == 0) return 0;
    hipLaunchKernelGGL(k_block_norm_sums, dim3((b.f.D + NORM_SUM_COLS - 1) / NORM_SUM_COLS, ny),
                       dim3(NORM_SUM_COLS * NORM_SUM_SLICES), 0, st, s, (int)grid.x, (int)grid.y);
    return mep_check_launch("mep_block_norm_bwd");
}
