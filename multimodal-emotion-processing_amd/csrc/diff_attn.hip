// mep_diff_attn_fwd / _bwd: differential attention.  With s_m = scale q_m k_m^T over the allowed keys (m = 1, 2),
//   A_m = softmax(s_m) (a row without an allowed key: zeros),  P = A_1 - lam A_2,  out = P v
// and backward with dP = dO v^T, D_m = sum_k A_m dP:
//   dS_1 = A_1 (dP - D_1), dS_2 = -lam A_2 (dP - D_2), dq_m = scale dS_m k_m, dk_m = scale dS_m^T q_m, dv = P^T dO, dlam = -D_2.
//
// The rows of a (batch, key head) are its Tq queries times the H / G heads that share the key head, query-major: row r is
// query r / n of head n * g + r % n, so shared heads read one copy of the keys and their gradients are summed in registers.
//
// The difference is formed before anything is rounded to 16 bits: two nearly equal maps cancel, and rounding each of them
// first would leave an error of 2^-9 of the parts in a difference of a few hundredths.  That takes both rows' maxima and
// sums in advance, so the forward reads the keys twice: pass 1 for the statistics (online, each lane over its own keys, joined
// once at the end), pass 2 for P and P v.  Scores, statistics and accumulators are fp32; P and dS are rounded once to the
// tensors' type as operands of the second products.
//
// Products on v_mfma_f32_32x32x16 (fp32: 32x32x2).  Scores are formed transposed (keys x rows): a lane holds one row and 16
// keys, the row statistics are lane-local, and the accumulator registers are the second product's operand as they are
// when its sum runs over the keys in the order {4h .. 4h+3, 8+4h .. 8+4h+3} of lane half h; the other operand (V^T, K^T, Q^T,
// dO^T) is read transposed from LDS by ds_read_b64_tr_b16 in that order.
#include "elem.h"

namespace {

using namespace mep;

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int DA_THREADS = 256, DA_WAVES = 4, DA_ROWS = 32 * DA_WAVES;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float DA_MIN = -1.0e30f;      // the running maximum's start: finite, so that a row of masked keys stays 0 / 0-free

// One 16-byte operand of a lane: KS / 2 consecutive k of a 2 x (KS / 2) step, KS = 16 (8 in fp32)
template <int TYPE> struct Mat;
template <> struct Mat<MEP_BF16> {
    typedef __bf16 T;
    typedef __bf16 Frag __attribute__((ext_vector_type(8)));
    static constexpr int KS = 16, E = 8;
    static MEP_DEV floatx16 mma(Frag a, Frag b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<MEP_F16> {
    typedef _Float16 T;
    typedef _Float16 Frag __attribute__((ext_vector_type(8)));
    static constexpr int KS = 16, E = 8;
    static MEP_DEV floatx16 mma(Frag a, Frag b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<MEP_F32> {
    typedef float T;
    typedef f32x4 Frag;
    static constexpr int KS = 8, E = 4;
    static MEP_DEV floatx16 mma(Frag a, Frag b, floatx16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = mfma32(a[j], b[j], c);
        return c;
    }
};

// Geometry of an instance: head widths padded to DK (each map) and DV, LDS rows padded by one operand (16 bytes: the 32
// rows of an operand read then start in different banks)
template <int TYPE, int DK, int DV>
struct Geo {
    typedef Mat<TYPE> M;
    typedef typename M::T T;
    typedef typename M::Frag Frag;
    static constexpr int KT = TYPE == MEP_F32 ? 32 : 64;      // keys (or rows) of a staged tile
    static constexpr int KLD = 2 * DK + M::E, VLD = DV + M::E;
    static constexpr int NK = DK / M::KS, NV = DV / M::KS;    // operands along the head widths
    static constexpr int NP = 32 / M::KS;                     // operands of 32 keys
};

template <class M>
MEP_DEV typename M::Frag zero_frag() {
    typename M::Frag f;
#pragma unroll
    for (int j = 0; j < M::E; ++j) f[j] = (typename M::T)0.f;
    return f;
}

// E elements at column c of a row of n, zero behind it
template <class M>
MEP_DEV typename M::Frag row_frag(const MEP_G typename M::T* row, int c, int n, bool vec) {
    typename M::Frag f = zero_frag<M>();
    if (vec) {
        if (c < n) f = *reinterpret_cast<const MEP_G typename M::Frag*>(row + c);
    } else {
#pragma unroll
        for (int j = 0; j < M::E; ++j) if (c + j < n) f[j] = row[c + j];
    }
    return f;
}

// rows r of a tile with bit r of `valid` set, the others and the columns behind n as zeros (a masked key's contents, NaN
// too, never enter a product)
template <class M, int ROWS, int CP, int LD>
MEP_DEV void stage(typename M::T* dst, const MEP_G typename M::T* src, int64_t ld, int n, bool vec, unsigned long long valid) {
    constexpr int CH = CP / M::E;
    for (int i = threadIdx.x; i < ROWS * CH; i += DA_THREADS) {
        const int r = i / CH, c = i % CH * M::E;
        typename M::Frag f = zero_frag<M>();
        if (valid >> r & 1) f = row_frag<M>(src + r * ld, c, n, vec);
        *reinterpret_cast<typename M::Frag*>(dst + r * LD + c) = f;
    }
}

// first-product operand: row (lane & 31), elements KS i + E h ..
template <class M>
MEP_DEV typename M::Frag lds_frag(const typename M::T* tile, int ld, int i) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const typename M::Frag*>(tile + (lane & 31) * ld + M::KS * i + M::E * (lane >> 5));
}

// second-product operand: column 32 n + (lane & 31) of the tile, the rows of step i in accumulator order
template <class M>
MEP_DEV typename M::Frag lds_frag_t(const typename M::T* tile, int ld, int i, int n) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (M::KS == 8) {
        typename M::Frag f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = tile[(8 * i + 4 * h + j) * ld + 32 * n + (lane & 31)];
        return f;
    } else {
        // the 16 lanes of a group read 4 rows x 16 columns and get a column's 4 rows each
        const typename M::T* p = tile + (16 * i + 4 * h + ((lane & 15) >> 2)) * ld + 32 * n + (lane & 16) + 4 * (lane & 3);
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * ld));
        return __builtin_bit_cast(typename M::Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// an accumulator tile as operand i of the next product, rounded to the tensors' type
template <class M>
MEP_DEV typename M::Frag acc_frag(const floatx16& p, int i) {
    typename M::Frag f;
#pragma unroll
    for (int j = 0; j < M::E; ++j) f[j] = (typename M::T)p[M::E * i + j];
    return f;
}

MEP_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
MEP_DEV float half_swap(float v) { return __shfl_xor(v, 32); }

// what a workgroup works on, and its keys
struct Job {
    int b, g, block, n;          // batch row, key head, block of rows or keys, heads per key head
    int rows, len, first;        // Tq n; allowed keys are below len; causal: key <= first + query
};
MEP_DEV Job make_job(const mep_diff_attn_desc& d, int blocks, bool reverse) {
    Job j;
    const int bg = blockIdx.x / blocks;
    j.block = blockIdx.x - bg * blocks;
    if (reverse) j.block = blocks - 1 - j.block;      // causal: the longest blocks start first
    j.b = bg / d.G;
    j.g = bg - j.b * d.G;
    j.n = d.H / d.G;
    j.rows = d.Tq * j.n;
    j.len = d.Tk;
    if (d.lengths) j.len = max(0, min(j.len, G<const int>(d.lengths)[j.b]));
    j.first = d.Tk - d.Tq;
    if (d.q_start) j.first = max(-(1 << 30), min(1 << 30, G<const int>(d.q_start)[j.b]));
    if (d.causal) j.len = max(0, min(j.len, j.first + d.Tq));     // what no query sees is never read
    return j;
}
// keys that any of the queries up to t may see
MEP_DEV int key_end(const mep_diff_attn_desc& d, const Job& j, int t) {
    return d.causal ? max(0, min(j.len, j.first + t + 1)) : j.len;
}

MEP_DEV bool mask_at(const mep_diff_attn_desc& d, int64_t o) {
    return d.mask_float ? G<const float>(d.mask)[o] != 0.f : G<const uint8_t>(d.mask)[o] != 0;
}
// bit i: key k0 + i of the tile is there and not masked for every query
MEP_DEV unsigned long long key_bits(const mep_diff_attn_desc& d, const Job& j, int k0, int n) {
    const int i = threadIdx.x & 63, k = k0 + i;
    bool on = i < n && k < j.len;
    if (on && d.mask_form == 1) on = mask_at(d, (int64_t)j.b * d.m_sB + (int64_t)k * d.m_sK);
    return __ballot(on);
}
// a tile position in accumulator order: acc_row(r, lane) = acc_off(r) + 4 h
MEP_DEV constexpr int acc_off(int r) { return (r & 3) + 8 * (r >> 2); }

// scores of keys k0 .. k0 + 31 (rows of the accumulator) against this lane's query t: masked ones to -inf
MEP_DEV void mask_keys(const mep_diff_attn_desc& d, const Job& j, int k0, unsigned bits, int t, floatx16& s1, floatx16& s2) {
    const int h = (threadIdx.x & 63) >> 5;
    unsigned on = bits >> (4 * h);
    if (d.causal) {      // keys up to first + t
        const int last = j.first + t - k0 - 4 * h;
        on &= last < 0 ? 0u : last > 30 ? ~0u : (2u << last) - 1u;
    }
    if (d.mask_form == 2) {
        const int64_t o = (int64_t)j.b * d.m_sB + (int64_t)t * d.m_sQ + (int64_t)(k0 + 4 * h) * d.m_sK;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if ((on >> acc_off(r) & 1) && !mask_at(d, o + (int64_t)acc_off(r) * d.m_sK)) on &= ~(1u << acc_off(r));
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const bool ok = on >> acc_off(r) & 1;
        s1[r] = ok ? s1[r] : -INFINITY;
        s2[r] = ok ? s2[r] : -INFINITY;
    }
}

// One row's two softmax statistics: the scaled maximum m (log2 units) and 1 / sum of 2^(s c - m).  They are kept apart: a
// single logarithm of the sum loses the low bits of m when the scores are large.
struct RowStat { float m1, i1, m2, i2; };

// ------------------------------------------------------------------ forward
template <int TYPE, int DK, int DV>
__global__ __launch_bounds__(DA_THREADS) void k_diff_fwd(mep_diff_attn_desc d, int blocks) {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    constexpr int KT = Ge::KT, KLD = Ge::KLD, VLD = Ge::VLD;
    __shared__ __align__(16) T Ks[KT * KLD];
    __shared__ __align__(16) T Vs[KT * VLD];
    const Job j = make_job(d, blocks, d.causal);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int row0 = j.block * DA_ROWS + wave * 32, row = row0 + (lane & 31);
    const bool live = row < j.rows;
    const int rr = live ? row : j.rows - 1, t = rr / j.n, head = j.g * j.n + rr - t * j.n;
    const bool vq = d.vec & 1, vk = d.vec & 2, vv = d.vec & 4;
    const float c = d.scale * LOG2E;

    Frag q[2][Ge::NK];
    {
        const MEP_G T* qp = G<const T>(d.q) + (int64_t)j.b * d.q_sB + (int64_t)t * d.q_sT + (int64_t)head * d.q_sH;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < Ge::NK; ++i)
                q[m][i] = live ? row_frag<M>(qp + m * d.q_sM, M::KS * i + M::E * h, d.d, vq) : zero_frag<M>();
    }
    const MEP_G T* kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH;
    const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH;
    const int tlast = (min(j.rows, (j.block + 1) * DA_ROWS) - 1) / j.n;      // the block's last query
    const int end = key_end(d, j, tlast);
    const int wend = row0 < j.rows ? key_end(d, j, (min(j.rows, row0 + 32) - 1) / j.n) : 0;   // the wave's
    const int wfull = d.causal ? j.first + row0 / j.n + 1 : INT_MAX;         // keys below are causal for all its rows

    auto scores = [&](int sub, int k0, unsigned bits, floatx16& s1, floatx16& s2) {
        s1 = zero16();
        s2 = zero16();
        const T* kt = Ks + 32 * sub * KLD;
#pragma unroll
        for (int i = 0; i < Ge::NK; ++i) {
            s1 = M::mma(lds_frag<M>(kt, KLD, i), q[0][i], s1);
            s2 = M::mma(lds_frag<M>(kt + DK, KLD, i), q[1][i], s2);
        }
        if (bits != ~0u || k0 + 32 > wfull || d.mask_form == 2) mask_keys(d, j, k0, bits, t, s1, s2);
    };

    // pass 1: the statistics
    RowStat st = {DA_MIN * c, 0.f, DA_MIN * c, 0.f};
    auto online = [&](const floatx16& s, float& m, float& l) {
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        const float mn = fmaxf(m, mx * c);
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += exp2_fast(fmaf(s[r], c, -mn));
        l = fmaf(l, exp2_fast(m - mn), sum);
        m = mn;
    };
    for (int k0 = 0; k0 < end; k0 += KT) {
        const unsigned long long bits = key_bits(d, j, k0, KT);
        __syncthreads();
        stage<M, KT, DK, KLD>(Ks, kp + k0 * d.k_sT, d.k_sT, d.d, vk, bits);
        stage<M, KT, DK, KLD>(Ks + DK, kp + k0 * d.k_sT + d.k_sM, d.k_sT, d.d, vk, bits);
        __syncthreads();
#pragma unroll
        for (int sub = 0; sub < KT / 32; ++sub) {
            const int ks = k0 + 32 * sub;
            if (ks >= wend) break;
            floatx16 s1, s2;
            scores(sub, ks, (unsigned)(bits >> (32 * sub)), s1, s2);
            online(s1, st.m1, st.i1);
            online(s2, st.m2, st.i2);
        }
    }
    // join the two halves of each row's keys, and invert the sums (0 for a row without keys)
    auto join = [&](float& m, float& l) {
        const float mo = half_swap(m), lo = half_swap(l), mn = fmaxf(m, mo);
        l = l * exp2_fast(m - mn) + lo * exp2_fast(mo - mn);
        l = l > 0.f ? 1.0f / l : (l == l ? 0.f : l);
        m = mn;
    };
    join(st.m1, st.i1);
    join(st.m2, st.i2);
    if (d.stats && live && h == 0)
        *reinterpret_cast<MEP_G f32x4*>(G<float>(d.stats) + 4 * (((int64_t)j.b * d.H + head) * d.Tq + t)) = f32x4{st.m1, st.i1, st.m2, st.i2};
    const float lam = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)t * d.lam_sT + (int64_t)head * d.lam_sH];
    // P is formed times rho, so that neither map's factor is over 1 nor both are small: of 1 / sum's size, a float16 operand
    // would be subnormal over long rows.  (A row without keys has both factors 0.)
    const float both = fmaxf(st.i1, fabsf(lam * st.i2)), rho = both > 0.f ? 1.0f / both : 0.f;
    const float f1 = st.i1 * rho, f2 = lam * st.i2 * rho;

    // pass 2: P and P v, transposed (the value channels are the accumulator's rows)
    floatx16 o[DV / 32];
#pragma unroll
    for (int n = 0; n < DV / 32; ++n) o[n] = zero16();
    for (int k0 = 0; k0 < end; k0 += KT) {
        const unsigned long long bits = key_bits(d, j, k0, KT);
        __syncthreads();
        stage<M, KT, DK, KLD>(Ks, kp + k0 * d.k_sT, d.k_sT, d.d, vk, bits);
        stage<M, KT, DK, KLD>(Ks + DK, kp + k0 * d.k_sT + d.k_sM, d.k_sT, d.d, vk, bits);
        stage<M, KT, DV, VLD>(Vs, vp + k0 * d.v_sT, d.v_sT, d.dv, vv, bits);
        __syncthreads();
#pragma unroll
        for (int sub = 0; sub < KT / 32; ++sub) {
            const int ks = k0 + 32 * sub;
            if (ks >= wend) break;
            floatx16 s1, s2;
            scores(sub, ks, (unsigned)(bits >> (32 * sub)), s1, s2);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s1[r] = exp2_fast(fmaf(s1[r], c, -st.m1)) * f1 - f2 * exp2_fast(fmaf(s2[r], c, -st.m2));
#pragma unroll
            for (int i = 0; i < Ge::NP; ++i) {
                const Frag p = acc_frag<M>(s1, i);
#pragma unroll
                for (int n = 0; n < DV / 32; ++n) o[n] = M::mma(lds_frag_t<M>(Vs + 32 * sub * VLD, VLD, i, n), p, o[n]);
            }
        }
    }
    if (live) {
        MEP_G T* out = G<T>(d.out) + (((int64_t)j.b * d.Tq + t) * d.H + head) * d.dv;
#pragma unroll
        for (int n = 0; n < DV / 32; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = 32 * n + acc_off(r) + 4 * h;
                if (col < d.dv) out[col] = (T)(o[n][r] * both);
            }
    }
}

// ------------------------------------------------------------------ backward: D and dq
template <int TYPE, int DK, int DV>
__global__ __launch_bounds__(DA_THREADS) void k_diff_bwd_q(mep_diff_attn_bwd_desc bd, int blocks) {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    constexpr int KT = Ge::KT, KLD = Ge::KLD, VLD = Ge::VLD;
    const mep_diff_attn_desc& d = bd.f;
    __shared__ __align__(16) T Ks[KT * KLD];
    __shared__ __align__(16) T Vs[KT * VLD];
    const Job j = make_job(d, blocks, d.causal);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int row0 = j.block * DA_ROWS + wave * 32, row = row0 + (lane & 31);
    const bool live = row < j.rows;
    const int rr = live ? row : j.rows - 1, t = rr / j.n, head = j.g * j.n + rr - t * j.n;
    const bool vq = d.vec & 1, vk = d.vec & 2, vv = d.vec & 4, vo = d.vec & 8;
    const float c = d.scale * LOG2E;

    Frag q[2][Ge::NK], g[Ge::NV];
    {
        const MEP_G T* qp = G<const T>(d.q) + (int64_t)j.b * d.q_sB + (int64_t)t * d.q_sT + (int64_t)head * d.q_sH;
        const MEP_G T* gp = G<const T>(bd.dout) + (int64_t)j.b * bd.o_sB + (int64_t)t * bd.o_sT + (int64_t)head * bd.o_sH;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < Ge::NK; ++i)
                q[m][i] = live ? row_frag<M>(qp + m * d.q_sM, M::KS * i + M::E * h, d.d, vq) : zero_frag<M>();
#pragma unroll
        for (int i = 0; i < Ge::NV; ++i) g[i] = live ? row_frag<M>(gp, M::KS * i + M::E * h, d.dv, vo) : zero_frag<M>();
    }
    const MEP_G T* kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH;
    const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH;
    const int64_t srow = ((int64_t)j.b * d.H + head) * d.Tq + t;
    const f32x4 sv = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(d.stats) + 4 * srow);
    const RowStat st = {sv[0], sv[1], sv[2], sv[3]};
    const float lam = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)t * d.lam_sT + (int64_t)head * d.lam_sH];
    const int tlast = (min(j.rows, (j.block + 1) * DA_ROWS) - 1) / j.n;
    const int end = key_end(d, j, tlast);
    const int wend = row0 < j.rows ? key_end(d, j, (min(j.rows, row0 + 32) - 1) / j.n) : 0;
    const int wfull = d.causal ? j.first + row0 / j.n + 1 : INT_MAX;

    // s1, s2 become 2^(s c - m): A_m without its 1 / sum
    auto maps = [&](int sub, int k0, unsigned bits, floatx16& s1, floatx16& s2, floatx16& dp) {
        s1 = zero16();
        s2 = zero16();
        dp = zero16();
        const T* kt = Ks + 32 * sub * KLD;
#pragma unroll
        for (int i = 0; i < Ge::NK; ++i) {
            s1 = M::mma(lds_frag<M>(kt, KLD, i), q[0][i], s1);
            s2 = M::mma(lds_frag<M>(kt + DK, KLD, i), q[1][i], s2);
        }
#pragma unroll
        for (int i = 0; i < Ge::NV; ++i) dp = M::mma(lds_frag<M>(Vs + 32 * sub * VLD, VLD, i), g[i], dp);
        if (bits != ~0u || k0 + 32 > wfull || d.mask_form == 2) mask_keys(d, j, k0, bits, t, s1, s2);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s1[r] = exp2_fast(fmaf(s1[r], c, -st.m1));
            s2[r] = exp2_fast(fmaf(s2[r], c, -st.m2));
        }
    };
    float d1 = 0.f, d2 = 0.f;
    floatx16 a[2][DK / 32];
#pragma unroll
    for (int n = 0; n < DK / 32; ++n) a[0][n] = a[1][n] = zero16();
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        for (int k0 = 0; k0 < end; k0 += KT) {
            const unsigned long long bits = key_bits(d, j, k0, KT);
            __syncthreads();
            stage<M, KT, DK, KLD>(Ks, kp + k0 * d.k_sT, d.k_sT, d.d, vk, bits);
            stage<M, KT, DK, KLD>(Ks + DK, kp + k0 * d.k_sT + d.k_sM, d.k_sT, d.d, vk, bits);
            stage<M, KT, DV, VLD>(Vs, vp + k0 * d.v_sT, d.v_sT, d.dv, vv, bits);
            __syncthreads();
#pragma unroll
            for (int sub = 0; sub < KT / 32; ++sub) {
                const int ks = k0 + 32 * sub;
                if (ks >= wend) break;
                floatx16 s1, s2, dp;
                maps(sub, ks, (unsigned)(bits >> (32 * sub)), s1, s2, dp);
                if (pass == 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        d1 = fmaf(s1[r], dp[r], d1);
                        d2 = fmaf(s2[r], dp[r], d2);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        s1[r] *= dp[r] - d1;       // dS_m without the row's factors i1, -lam i2
                        s2[r] *= dp[r] - d2;
                    }
                    const T* kt = Ks + 32 * sub * KLD;
#pragma unroll
                    for (int i = 0; i < Ge::NP; ++i) {
                        const Frag f1 = acc_frag<M>(s1, i), f2 = acc_frag<M>(s2, i);
#pragma unroll
                        for (int n = 0; n < DK / 32; ++n) {
                            a[0][n] = M::mma(lds_frag_t<M>(kt, KLD, i, n), f1, a[0][n]);
                            a[1][n] = M::mma(lds_frag_t<M>(kt + DK, KLD, i, n), f2, a[1][n]);
                        }
                    }
                }
            }
        }
        if (pass == 0) {
            d1 = (d1 + half_swap(d1)) * st.i1;
            d2 = (d2 + half_swap(d2)) * st.i2;
            if (live && h == 0) {
                G<float>(bd.delta)[2 * srow] = d1;
                G<float>(bd.delta)[2 * srow + 1] = d2;
                if (bd.dlam_rows) G<float>(bd.dlam_rows)[((int64_t)j.b * d.Tq + t) * d.H + head] = -d2;
            }
        }
    }
    if (live && bd.dq) {
        MEP_G T* out = G<T>(bd.dq) + (((int64_t)j.b * d.Tq + t) * d.H + head) * 2 * d.d;
        const float f[2] = {st.i1 * d.scale, -lam * st.i2 * d.scale};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < DK / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int col = 32 * n + acc_off(r) + 4 * h;
                    if (col < d.d) out[m * d.d + col] = (T)(a[m][n][r] * f[m]);
                }
    }
}

// ------------------------------------------------------------------ backward: dk and dv
// A wave owns 32 keys (an accumulator column each) and walks the rows; KREG: its K and V operands stay in registers.
template <int TYPE, int DK, int DV, bool KREG>
__global__ __launch_bounds__(DA_THREADS) void k_diff_bwd_kv(mep_diff_attn_bwd_desc bd, int blocks) {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    constexpr int RT = Ge::KT, QLD = Ge::KLD, OLD = Ge::VLD;
    const mep_diff_attn_desc& d = bd.f;
    __shared__ __align__(16) T Qs[RT * QLD];
    __shared__ __align__(16) T Os[RT * OLD];
    __shared__ __align__(16) float Rs[6][RT];      // a row's m1, m2, i1, lam i2, i1 D1, lam i2 D2
    __shared__ int Ts[RT];                         // and its query
    const Job j = make_job(d, blocks, false);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int key0 = j.block * DA_ROWS + wave * 32, key = key0 + (lane & 31);
    const bool vq = d.vec & 1, vk = d.vec & 2, vv = d.vec & 4, vo = d.vec & 8;
    const float c = d.scale * LOG2E;
    bool on = key < j.len;
    if (on && d.mask_form == 1) on = mask_at(d, (int64_t)j.b * d.m_sB + (int64_t)key * d.m_sK);
    const MEP_G T* kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH + (int64_t)(on ? key : 0) * d.k_sT;
    const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH + (int64_t)(on ? key : 0) * d.v_sT;
    auto load_k = [&](int m, int i) { return on ? row_frag<M>(kp + m * d.k_sM, M::KS * i + M::E * h, d.d, vk) : zero_frag<M>(); };
    auto load_v = [&](int i) { return on ? row_frag<M>(vp, M::KS * i + M::E * h, d.dv, vv) : zero_frag<M>(); };
    Frag kr[2][KREG ? Ge::NK : 1], vr[KREG ? Ge::NV : 1];
    if constexpr (KREG) {
#pragma unroll
        for (int i = 0; i < Ge::NK; ++i) { kr[0][i] = load_k(0, i); kr[1][i] = load_k(1, i); }
#pragma unroll
        for (int i = 0; i < Ge::NV; ++i) vr[i] = load_v(i);
    }
    floatx16 ak[2][DK / 32], av[DV / 32];
#pragma unroll
    for (int n = 0; n < DK / 32; ++n) ak[0][n] = ak[1][n] = zero16();
#pragma unroll
    for (int n = 0; n < DV / 32; ++n) av[n] = zero16();
    // rows that see any of the block's / the wave's keys; every one of the wave's keys: from row wfull on
    const int bstart = d.causal ? max(0, min(d.Tq, j.block * DA_ROWS - j.first)) * j.n : 0;
    const int wstart = d.causal ? max(0, min(d.Tq, key0 - j.first)) * j.n : 0;
    const int wfull = d.causal ? max(0, min(d.Tq, key0 + 31 - j.first)) * j.n : 0;
    const bool wave_on = __ballot(on) != 0, all_on = __ballot(on) == ~0ull;
    const int rend = j.block * DA_ROWS < j.len ? j.rows : 0;

    for (int r0 = bstart / RT * RT; r0 < rend; r0 += RT) {
        __syncthreads();
        {
            const MEP_G T* qb = G<const T>(d.q) + (int64_t)j.b * d.q_sB;
            const MEP_G T* ob = G<const T>(bd.dout) + (int64_t)j.b * bd.o_sB;
            constexpr int CQ = DK / M::E, CO = DV / M::E, CH = 2 * CQ + CO;
            for (int i = threadIdx.x; i < RT * CH; i += DA_THREADS) {
                const int r = i / CH, ch = i % CH, row = r0 + r;
                const int t = min(row, j.rows - 1) / j.n, head = j.g * j.n + min(row, j.rows - 1) - t * j.n;
                Frag f = zero_frag<M>();
                if (ch < 2 * CQ) {
                    const int m = ch / CQ, col = ch % CQ * M::E;
                    if (row < j.rows) f = row_frag<M>(qb + (int64_t)t * d.q_sT + (int64_t)head * d.q_sH + m * d.q_sM, col, d.d, vq);
                    *reinterpret_cast<Frag*>(Qs + r * QLD + m * DK + col) = f;
                } else {
                    const int col = (ch - 2 * CQ) * M::E;
                    if (row < j.rows) f = row_frag<M>(ob + (int64_t)t * bd.o_sT + (int64_t)head * bd.o_sH, col, d.dv, vo);
                    *reinterpret_cast<Frag*>(Os + r * OLD + col) = f;
                }
            }
            if (threadIdx.x < RT) {
                const int row = r0 + threadIdx.x;
                float m1 = 0.f, m2 = 0.f, i1 = 0.f, li2 = 0.f, w1 = 0.f, w2 = 0.f;     // a row past the end: A = 0
                int t = 0;
                if (row < j.rows) {
                    t = row / j.n;
                    const int head = j.g * j.n + row - t * j.n;
                    const int64_t srow = ((int64_t)j.b * d.H + head) * d.Tq + t;
                    const f32x4 sv = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(d.stats) + 4 * srow);
                    const float lam = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)t * d.lam_sT + (int64_t)head * d.lam_sH];
                    m1 = sv[0]; i1 = sv[1]; m2 = sv[2]; li2 = lam * sv[3];
                    w1 = i1 * G<const float>(bd.delta)[2 * srow];
                    w2 = li2 * G<const float>(bd.delta)[2 * srow + 1];
                }
                Rs[0][threadIdx.x] = m1; Rs[1][threadIdx.x] = m2; Rs[2][threadIdx.x] = i1;
                Rs[3][threadIdx.x] = li2; Rs[4][threadIdx.x] = w1; Rs[5][threadIdx.x] = w2;
                Ts[threadIdx.x] = t;
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int sub = 0; sub < RT / 32; ++sub) {
            const int rs = r0 + 32 * sub;
            if (!wave_on || rs >= j.rows || rs + 32 <= wstart) continue;
            floatx16 s1 = zero16(), s2 = zero16(), dp = zero16();
            const T* qt = Qs + 32 * sub * QLD;
            const T* ot = Os + 32 * sub * OLD;
#pragma unroll
            for (int i = 0; i < Ge::NK; ++i) {
                const Frag k1 = KREG ? kr[0][KREG ? i : 0] : load_k(0, i), k2 = KREG ? kr[1][KREG ? i : 0] : load_k(1, i);
                s1 = M::mma(lds_frag<M>(qt, QLD, i), k1, s1);
                s2 = M::mma(lds_frag<M>(qt + DK, QLD, i), k2, s2);
            }
#pragma unroll
            for (int i = 0; i < Ge::NV; ++i) {
                const Frag v = KREG ? vr[KREG ? i : 0] : load_v(i);
                dp = M::mma(lds_frag<M>(ot, OLD, i), v, dp);
            }
            const bool partial = !all_on || rs < wfull || d.mask_form == 2;
            floatx16 p;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int lr = 32 * sub + acc_off(r) + 4 * h;
                float x1 = s1[r], x2 = s2[r];
                if (partial) {
                    const int t = Ts[lr];
                    bool ok = on && (!d.causal || key <= j.first + t);
                    if (ok && d.mask_form == 2) ok = mask_at(d, (int64_t)j.b * d.m_sB + (int64_t)t * d.m_sQ + (int64_t)key * d.m_sK);
                    x1 = ok ? x1 : -INFINITY;
                    x2 = ok ? x2 : -INFINITY;
                }
                x1 = exp2_fast(fmaf(x1, c, -Rs[0][lr]));
                x2 = exp2_fast(fmaf(x2, c, -Rs[1][lr]));
                p[r] = x1 * Rs[2][lr] - x2 * Rs[3][lr];
                s1[r] = x1 * fmaf(dp[r], Rs[2][lr], -Rs[4][lr]);
                s2[r] = x2 * fmaf(dp[r], -Rs[3][lr], Rs[5][lr]);
            }
#pragma unroll
            for (int i = 0; i < Ge::NP; ++i) {
                const Frag fp = acc_frag<M>(p, i), f1 = acc_frag<M>(s1, i), f2 = acc_frag<M>(s2, i);
#pragma unroll
                for (int n = 0; n < DV / 32; ++n) av[n] = M::mma(lds_frag_t<M>(ot, OLD, i, n), fp, av[n]);
#pragma unroll
                for (int n = 0; n < DK / 32; ++n) {
                    ak[0][n] = M::mma(lds_frag_t<M>(qt, QLD, i, n), f1, ak[0][n]);
                    ak[1][n] = M::mma(lds_frag_t<M>(qt + DK, QLD, i, n), f2, ak[1][n]);
                }
            }
        }
    }
    if (key < d.Tk) {      // masked keys and keys past the lengths get zeros
        MEP_G T* ok = G<T>(bd.dk) + (((int64_t)j.b * d.Tk + key) * d.G + j.g) * 2 * d.d;
        MEP_G T* ov = G<T>(bd.dv) + (((int64_t)j.b * d.Tk + key) * d.G + j.g) * d.dv;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < DK / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int col = 32 * n + acc_off(r) + 4 * h;
                    if (col < d.d) ok[m * d.d + col] = (T)(ak[m][n][r] * d.scale);
                }
#pragma unroll
        for (int n = 0; n < DV / 32; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = 32 * n + acc_off(r) + 4 * h;
                if (col < d.dv) ov[col] = (T)av[n][r];
            }
    }
}

// dlam[h] = -sum of D2 over batch and queries, in a fixed order
__global__ __launch_bounds__(DA_THREADS) void k_diff_dlam(mep_diff_attn_bwd_desc bd) {
    const mep_diff_attn_desc& d = bd.f;
    __shared__ float part[DA_WAVES];
    const int h = blockIdx.x;
    float s = 0.f;
    for (int b = 0; b < d.B; ++b) {
        const gfloat* p = G<const float>(bd.delta) + 2 * ((int64_t)b * d.H + h) * d.Tq;
        for (int t = threadIdx.x; t < d.Tq; t += DA_THREADS) s -= p[2 * (int64_t)t + 1];
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) G<float>(bd.dlam)[h] = (part[0] + part[1]) + (part[2] + part[3]);
}

// ------------------------------------------------------------------ host
enum { RUN_FWD, RUN_BWD_Q, RUN_BWD_KV };

template <int TYPE, int DK, int DV>
void run_instance(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, hipStream_t st) {
    // fp32 keys of 128 + 128 + 256 channels beside their gradients' accumulators would need more than the register file
    constexpr bool KREG = !(TYPE == MEP_F32 && DK >= 128);
    if (what == RUN_FWD) hipLaunchKernelGGL((k_diff_fwd<TYPE, DK, DV>), dim3(grid), dim3(DA_THREADS), 0, st, d, blocks);
    else if (what == RUN_BWD_Q) hipLaunchKernelGGL((k_diff_bwd_q<TYPE, DK, DV>), dim3(grid), dim3(DA_THREADS), 0, st, *b, blocks);
    else hipLaunchKernelGGL((k_diff_bwd_kv<TYPE, DK, DV, KREG>), dim3(grid), dim3(DA_THREADS), 0, st, *b, blocks);
}

template <int TYPE>
void pick_widths(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, hipStream_t st) {
    if (d.d <= 32 && d.dv <= 32) run_instance<TYPE, 32, 32>(what, d, b, grid, blocks, st);
    else if (d.d <= 32 && d.dv <= 64) run_instance<TYPE, 32, 64>(what, d, b, grid, blocks, st);
    else if (d.d <= 64 && d.dv <= 64) run_instance<TYPE, 64, 64>(what, d, b, grid, blocks, st);
    else if (d.d <= 64 && d.dv <= 128) run_instance<TYPE, 64, 128>(what, d, b, grid, blocks, st);
    else if (d.dv <= 128) run_instance<TYPE, 128, 128>(what, d, b, grid, blocks, st);
    else run_instance<TYPE, 128, 256>(what, d, b, grid, blocks, st);
}

// 16-byte operands can be read from rows of these strides
bool vec_rows(uint64_t p, int es, int n, int64_t a, int64_t b, int64_t c, int64_t e) {
    const int V = 16 / es;
    return p % 16 == 0 && n % V == 0 && a % V == 0 && b % V == 0 && c % V == 0 && e % V == 0;
}

// fills d.vec; the workgroups of a launch over `items` rows or keys per (batch, key head), or -1 (too many)
int64_t plan(mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, int64_t items, int& blocks) {
    const int es = d.type == MEP_F32 ? 4 : 2;
    d.vec = (vec_rows(d.q, es, d.d, d.q_sB, d.q_sT, d.q_sH, d.q_sM) ? 1 : 0) | (vec_rows(d.k, es, d.d, d.k_sB, d.k_sT, d.k_sH, d.k_sM) ? 2 : 0) |
            (vec_rows(d.v, es, d.dv, d.v_sB, d.v_sT, d.v_sH, 0) ? 4 : 0) |
            (b && vec_rows(b->dout, es, d.dv, b->o_sB, b->o_sT, b->o_sH, 0) ? 8 : 0);
    blocks = (int)((items + DA_ROWS - 1) / DA_ROWS);
    const int64_t grid = (int64_t)blocks * d.B * d.G;
    return grid * DA_THREADS < ((int64_t)1 << 32) ? grid : -1;
}

void run(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, int64_t grid, int blocks, hipStream_t st) {
    if (d.type == MEP_F32) pick_widths<MEP_F32>(what, d, b, (unsigned)grid, blocks, st);
    else if (d.type == MEP_BF16) pick_widths<MEP_BF16>(what, d, b, (unsigned)grid, blocks, st);
    else pick_widths<MEP_F16>(what, d, b, (unsigned)grid, blocks, st);
}

bool attn_ok(const mep_diff_attn_desc& d) {
    if (d.B < 0 || d.Tq < 0 || d.Tk < 0 || d.H < 1 || d.G < 1 || d.H % d.G || d.type < MEP_F32 || d.type > MEP_F16) return false;
    if (d.d < 1 || d.d > MEP_DIFF_ATTN_MAX_D || d.dv < 1 || d.dv > MEP_DIFF_ATTN_MAX_DV) return false;
    if (d.Tk >= 1 << 30 || (int64_t)d.Tq * (d.H / d.G) >= 1 << 30) return false;
    if (!(d.scale > 0.f && d.scale <= 1e6f) || d.mask_form < 0 || d.mask_form > 2 || (d.mask_form != 0) != (d.mask != 0)) return false;
    const bool empty = d.B == 0 || d.Tq == 0;
    return empty || (d.q && d.lam && d.out && (d.Tk == 0 || (d.k && d.v)));
}

}  // namespace

extern "C" int mep_diff_attn_fwd(const mep_diff_attn_desc* desc, mep_stream_t stream) {
    if (!desc || !attn_ok(*desc)) { mep_set_error("mep_diff_attn_fwd: invalid descriptor"); return MEP_EINVAL; }
    mep_diff_attn_desc d = *desc;
    if (d.B == 0 || d.Tq == 0) return 0;
    int blocks;
    const int64_t grid = plan(d, nullptr, (int64_t)d.Tq * (d.H / d.G), blocks);
    if (grid < 0) { mep_set_error("mep_diff_attn_fwd: too many rows for one launch"); return MEP_EINVAL; }
    run(RUN_FWD, d, nullptr, grid, blocks, (hipStream_t)stream);
    return mep_check_launch("mep_diff_attn_fwd");
}

extern "C" int mep_diff_attn_bwd(const mep_diff_attn_bwd_desc* desc, mep_stream_t stream) {
    if (!desc || !attn_ok(desc->f)) { mep_set_error("mep_diff_attn_bwd: invalid descriptor"); return MEP_EINVAL; }
    mep_diff_attn_bwd_desc b = *desc;
    const mep_diff_attn_desc& d = b.f;
    const bool rows = d.B > 0 && d.Tq > 0, keys = d.B > 0 && d.Tk > 0;
    if ((rows && (!d.stats || !b.dout || !b.delta)) || (keys && (!b.dk != !b.dv))) {
        mep_set_error("mep_diff_attn_bwd: a missing operand");
        return MEP_EINVAL;
    }
    hipStream_t st = (hipStream_t)stream;
    int qb, kb;
    const int64_t qg = plan(b.f, &b, (int64_t)d.Tq * (d.H / d.G), qb), kg = plan(b.f, &b, d.Tk, kb);
    if (qg < 0 || kg < 0) { mep_set_error("mep_diff_attn_bwd: too many rows for one launch"); return MEP_EINVAL; }
    if (rows) run(RUN_BWD_Q, d, &b, qg, qb, st);
    if (keys && b.dk) run(RUN_BWD_KV, d, &b, kg, kb, st);
    if (b.dlam) hipLaunchKernelGGL(k_diff_dlam, dim3(d.H), dim3(DA_THREADS), 0, st, b);
    return mep_check_launch("mep_diff_attn_bwd");
}
