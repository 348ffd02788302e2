// Differential attention on the matrix cores (instantiated per element type in diff_attn_*.hip, entry points in diff_attn.hip).
// With s_m = scale q_m k_m^T over the allowed keys (m = 1, 2),
//   A_m = softmax(s_m) (a row without an allowed key: zeros),  P = A_1 - lam A_2,  out = P v
// and backward with dP = dO v^T, D_m = sum_k A_m dP = dO . (A_m v):
//   dS_1 = A_1 (dP - D_1), dS_2 = -lam A_2 (dP - D_2), dq_m = scale dS_m k_m, dk_m = scale dS_m^T q_m, dv = P^T dO, dlam = -D_2.
//
// The rows of a (batch, key head) are its Tq queries times the H / G heads that share the key head, query-major: row r is
// query r / n of head n * g + r % n, so shared heads read one copy of the keys and their gradients are summed in registers.
//
// The difference is formed before anything is rounded to 16 bits: two nearly equal maps cancel, and rounding each of them
// first would leave an error of 2^-9 of the parts in a difference of a few hundredths.  See k_diff_fwd for how one pass over the
// keys does that.  Scores, statistics and accumulators are fp32; P and dS are rounded once, as operands of the second products, because
// the matrix instructions take no wider ones.  In 16 bits results are so off by 1.4 times what rounding them alone would leave (whole
// errors of 2.3e-3 and 1.7e-3 in bf16, 2.9e-4 and 2.1e-4 in float16).
//
// Products on v_mfma_f32_32x32x16 (fp32: 32x32x2).  Scores are formed transposed (keys x rows): a lane holds one row and 16
// keys, the row statistics are lane-local, and the accumulator registers are the second product's operand as they are
// when its sum runs over the keys in the order {4h .. 4h+3, 8+4h .. 8+4h+3} of lane half h; the other operand (V^T, K^T, Q^T,
// dO^T) is read transposed from LDS by ds_read_b64_tr_b16 in that order.
//
// Tiles of 64 keys (32 in fp32) go to LDS by DMA, 16 bytes a lane, one tile ahead of the products, and are stored as 16-byte chunks
// whose place in the row is xor-ed with the row (Lay): both kinds of reads touch every bank equally often.
#pragma once
#include <climits>
#include <type_traits>

#include "elem.h"
#include "diff_order.h"

namespace mep {

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int DA_THREADS = 256, DA_WAVES = 4, DA_ROWS = 32 * DA_WAVES;
constexpr float DA_LOG2E = 1.4426950408889634f;
constexpr float DA_MIN = -1.0e30f;      // the running maximum's start: finite, so that masked scores (-inf) give 2^-inf = 0
constexpr unsigned DA_NOWHERE = 0x80000000u, DA_SPAN = 0x7fffffffu;   // a DMA offset behind the span reads zeros
enum { DA_FWD, DA_FWD_TWO, DA_SIZES, DA_BWD_Q, DA_BWD_Q_TWO, DA_BWD_KV, DA_SPLIT };

// keys of a tile of k_diff_split: 64 where two tiles fit 160 KB of LDS
constexpr int da_split_keys(int type, int dk, int dv) { return (type == MEP_F32 ? 4 : 2) * 2 * 64 * (2 * dk + dv) <= 160 * 1024 ? 64 : 32; }

// One 16-byte operand of a lane: E consecutive k of a 2 E step
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

// A tile of rows of COLS elements in LDS: chunk c (16 bytes) of row r lies at place c ^ sw(r) of the row.  sw differs over any
// 8 consecutive rows (first-product operands: the same chunk of 32 rows), and in pairs over any 4 (transposed reads:
// 2 neighbouring chunks of 4 rows).  Rows of 4 chunks share 128 bytes with their neighbour.
template <class M, int COLS>
struct Lay {
    static constexpr int CH = COLS / M::E;
    static_assert(CH == 4 || CH % 8 == 0, "row width");
    static MEP_DEV int sw(int r) { return CH >= 8 ? ((r & 3) << 1) | ((r >> 2) & 1) : (r & 2) | ((r >> 2) & 1); }
    static MEP_DEV int at(int r, int c) { return (r * CH + (c ^ sw(r))) * M::E; }
};

constexpr int da_piece(int width) { return width < 128 ? width : 128; }      // channels that pass through LDS at a time

// Geometry of an instance: head widths padded to DK (each map) and DV
template <int TYPE, int DK, int DV>
struct Geo {
    typedef Mat<TYPE> M;
    typedef typename M::T T;
    typedef typename M::Frag Frag;
    static constexpr int KT = TYPE == MEP_F32 ? 32 : 64;      // keys (or rows) of a staged tile
    static constexpr int NK = DK / M::KS, NV = DV / M::KS;    // operands along the head widths
    static constexpr int NP = 32 / M::KS;                     // operands of 32 keys
    static constexpr int STEP = 16 / M::KS;                   // operands of 16 channels
    static constexpr int KSZ = KT * 2 * DK, TSZ = KSZ + KT * DV;      // elements of a tile's keys, and of a tile
    static constexpr int OUT = DA_ROWS * (da_piece(DK > DV ? DK : DV) + M::E);  // the results pass through the tiles
    static constexpr int BUF = 2 * TSZ > OUT ? 2 * TSZ : OUT;
};

// Narrower heads than the instance: in fp32, whose products take 16 times as long, the products of 16 channels (of results: 32)
// behind a head's n are left out; in 16 bits the branches would cost more than the products
template <int TYPE>
MEP_DEV bool within(int col, int n) { return TYPE != MEP_F32 || col < n; }

template <class M>
MEP_DEV typename M::Frag zero_frag() {
    typename M::Frag f;
#pragma unroll
    for (int j = 0; j < M::E; ++j) f[j] = (typename M::T)0.f;
    return f;
}

// E elements at column c of a row of n (rows are padded to whole operands with zeros)
template <class M>
MEP_DEV typename M::Frag row_frag(const MEP_G typename M::T* row, int c, int n, bool live) {
    return live && c < n ? *reinterpret_cast<const MEP_G typename M::Frag*>(row + c) : zero_frag<M>();
}

// The N operands of a lane's row (n elements from p on): held in registers, or (wide fp32 heads, whose products take 16 times as long
// and whose operands and accumulators would not fit) read again from the cache at each use.  A row that is not there: zeros.
// One wave a SIMD with all its registers holds 64 channels of fp32, and two waves that read them again are slower (B 4, T 2048, 8
// heads, 64 / 128: forward 1366 us against 969, dk and dv 1787 against 1365), but for dq (64 / 64: 891 against 1048).
constexpr bool da_hold(int type, int dk) { return !(type == MEP_F32 && dk >= 128); }
constexpr bool da_hold_q(int type, int dk) { return !(type == MEP_F32 && dk >= 64); }
constexpr bool da_wide(int type, int dk) { return dk >= (type == MEP_F32 ? 64 : 128); }
template <class M, int N, bool HOLD>
struct Operand {
    typedef typename M::Frag Frag;
    Frag f[HOLD ? N : 1];
    const MEP_G typename M::T* p;
    int n;
    bool live;
    MEP_DEV Operand(const MEP_G typename M::T* row, int width, bool there) : p(row), n(width), live(there) {
        if constexpr (HOLD) {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = row_frag<M>(p, M::KS * i + M::E * ((threadIdx.x & 63) >> 5), n, live);
        }
    }
    MEP_DEV Frag at(int i) const {
        if constexpr (HOLD) {
            return f[i];
        } else {      // the load of a valid place without a branch, then the choice
            const int c = M::KS * i + M::E * ((threadIdx.x & 63) >> 5), last = (n - 1) / M::E * M::E;
            Frag x = *reinterpret_cast<const MEP_G Frag*>(p + min(c, last));
            const bool on = live && c < n;
#pragma unroll
            for (int e = 0; e < M::E; ++e) x[e] = on ? x[e] : (typename M::T)0.f;
            return x;
        }
    }
};

typedef __attribute__((address_space(3))) char da_lds_char;
typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes a lane from the buffer `rs` at off + soff to LDS at `dst` + 16 lane (dst of the wave).  In inline assembly, since the
// compiler would wait for every load in flight before the next LDS read, which is of the other tile; nothing but tile_sync
// waits for these.  The loads return no registers.  m0 is a reserved register, which the compiler keeps nothing in (it cannot be named
// as clobbered), and no other instruction of these kernels uses it.
MEP_DEV void dma16(const void* dst, unsigned off, i32x4 rs, unsigned soff) {
    const unsigned at = __builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)(const da_lds_char*)dst);
    soff = __builtin_amdgcn_readfirstlane((int)soff);
    // 5 wait states between a readfirstlane and a memory instruction that reads its result, 1 behind m0
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(off), "s"(rs), "s"(soff) : "memory");
}
// a raw buffer of DA_SPAN bytes from p on
MEP_DEV i32x4 da_buffer(const MEP_G void* p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)a), __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)), (int)DA_SPAN, 0x00020000};
}

// ROWS x COLS of LDS from rows of global memory, by DMA: an instruction of a wave fills 64 chunks, and instruction i of a
// lane takes chunk `chunk(i)` of row `row + i STEP`.  The chunk does not depend on i (with 4 or 2 rows a
// step, on i modulo 2 or 4 alone), so neither does the lane's offset, and a tile costs no address arithmetic: the row steps are the scalar offset.
template <class M, int ROWS, int COLS, int THREADS = DA_THREADS>
struct Stager {
    typedef Lay<M, COLS> L;
    typedef typename M::T T;
    static constexpr int STEP = THREADS / L::CH < ROWS ? THREADS / L::CH : ROWS, N = ROWS / STEP, NO = STEP % 8 ? 8 / STEP : 1;
    static constexpr bool ALL = STEP * L::CH == THREADS;      // else only the first waves load
    static_assert(STEP >= 2 && ROWS % STEP == 0, "tile");
    int row;
    unsigned off[NO];                // byte offset of the lane's chunk in row `row`, or DA_NOWHERE
    static MEP_DEV int chunk(int tid, int i) { return (tid % L::CH) ^ L::sw(tid / L::CH + i * STEP); }
    // where(c): element offset of chunk c within its row, or -1 where there is none
    template <class F>
    MEP_DEV Stager(int tid, unsigned stride, F where) {
        row = tid / L::CH;
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int o = where(chunk(tid, i));
            off[i] = o < 0 ? DA_NOWHERE : (unsigned)(row * stride + o) * (unsigned)sizeof(T);
        }
    }
    // rows of the tile with their bit set, `stride` elements apart from base on; zeros in the others.  Masked rows are never loaded:
    // their contents, NaN too, never enter a product.
    MEP_DEV void load(T* dst, const MEP_G T* base, unsigned stride, unsigned long long bits) const {
        const i32x4 rs = da_buffer(base);
        if (!ALL && threadIdx.x >= STEP * L::CH) return;
        const bool full = bits == (ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1);
        T* mine = dst + (threadIdx.x >> 6) * 64 * M::E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unsigned o = off[i % NO];
            if (!full && !(bits >> (row + i * STEP) & 1)) o = DA_NOWHERE;
            dma16(mine + i * THREADS * M::E, o, rs, i * STEP * stride * (unsigned)sizeof(T));
        }
    }
    // rows at any places: at(r): element offset of tile row r, or -1
    template <class F>
    MEP_DEV void gather(T* dst, const MEP_G T* base, unsigned stride, F at) const {
        if (!ALL && threadIdx.x >= STEP * L::CH) return;
        const i32x4 rs = da_buffer(base);
        T* mine = dst + (threadIdx.x >> 6) * 64 * M::E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int o = at(row + i * STEP);
            const unsigned c = off[i % NO];
            dma16(mine + i * THREADS * M::E, o < 0 || c == DA_NOWHERE ? DA_NOWHERE : c + (unsigned)(o - row * (int)stride) * (unsigned)sizeof(T), rs, 0);
        }
    }
};

// every wave's DMA and LDS accesses done, then the workgroup barrier
// (vmcnt = lgkmcnt = 0, by the builtin: the compiler then knows that nothing loaded before needs a wait behind it)
MEP_DEV void tile_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A lane's places in a tile.  a[j]: first-product operand, chunk 2 j + h of row lane & 31 (j = 0 .. 3 of a group of 8 chunks); the
// other rows and groups are constants away.  t[n]: second-product operand, in the rows of accumulator order and columns
// 32 n + (lane & 31), n = 0, 1; likewise (fp32: t[j], of row j of 4, any n).
template <class M, int COLS>
struct Reader {
    typedef Lay<M, COLS> L;
    typedef typename M::T T;
    typedef typename M::Frag Frag;
    static constexpr int NA = L::CH >= 8 ? 4 : 2, NT = M::KS == 8 ? 4 : L::CH >= 8 ? 2 : 1;
    int a[NA], t[NT];                // elements
    MEP_DEV Reader() {
        const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
        for (int j = 0; j < NA; ++j) a[j] = L::at(lane & 31, 2 * j + h);
        if constexpr (M::KS == 16) {     // the 16 lanes of a group read 4 rows x 16 columns and get a column's 4 rows each
#pragma unroll
            for (int n = 0; n < NT; ++n)
                t[n] = L::at(4 * h + ((lane & 15) >> 2), (32 * n + (lane & 16)) / M::E + ((lane & 3) >> 1)) + 4 * (lane & 1);
        } else {                         // row j of every 4
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = L::at(4 * h + j, (lane & 31) >> 2) + (lane & 3);
        }
    }
    // operand i (of all COLS) of the rows from r0 on
    MEP_DEV Frag rows(const T* tile, int r0, int i) const {
        return *reinterpret_cast<const Frag*>(tile + a[i % NA] + (r0 * L::CH + i / NA * 2 * NA) * M::E);
    }
    // step i of the rows from r0 on, columns col0 (a multiple of 32) ..
    MEP_DEV Frag cols(const T* tile, int r0, int col0, int i) const {
        if constexpr (M::KS == 8) {
            Frag f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = tile[t[j] + (r0 + 8 * i) * L::CH * M::E + col0];
            return f;
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const T* p = tile + t[col0 / 32 % NT] + ((r0 + 16 * i) * L::CH + col0 / (32 * NT) * (4 * NT)) * M::E;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * L::CH * M::E));
            return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// an accumulator tile as operand i of the next product, rounded to the tensors' type
template <class M>
MEP_DEV typename M::Frag acc_frag(const floatx16& p, int i) {
    typename M::Frag f;
#pragma unroll
    for (int j = 0; j < M::E; ++j) f[j] = (typename M::T)p[M::E * i + j];
    return f;
}

// (the instruction: off by 2^-23 of its result, as much as a score's own rounding)
MEP_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(s c - m), c = scale log2 e.  In fp32 the rounding of c is put right (it would shift every exponent the same way, by up to
// 2^-24 s c: a score's error would not average out); a masked score (-inf) stays one.  In 16 bits the operands' rounding is
// far above it.
template <int TYPE>
struct Exponent {
    float c, low;
    MEP_DEV explicit Exponent(float scale) {
        c = scale * DA_LOG2E;
        low = fmaf(scale, DA_LOG2E, -c) + scale * 1.9259629911e-8f;      // log2 e - DA_LOG2E
    }
    MEP_DEV float at(float s, float m) const {
        const float t = fmaf(s, c, -m);
        return exp2_fast(TYPE == MEP_F32 ? fmaf(fmaxf(s, DA_MIN), low, t) : t);
    }
};
// v over both lane halves of a row: lo and hi, each in every lane
MEP_DEV void both_halves(float v, float& lo, float& hi) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    lo = __builtin_bit_cast(float, a);
    hi = __builtin_bit_cast(float, b);
}
MEP_DEV float half_sum(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    return lo + hi;
}
MEP_DEV float half_max(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    return fmaxf(lo, hi);
}
MEP_DEV float max16(const floatx16& s) {
    float m = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
    return m;
}

// what a workgroup works on, and its keys
struct Job {
    int b, g, block, n;          // batch row, key head, block of rows or keys, heads per key head
    int rows, len, first;        // Tq n; allowed keys are below len; causal: key <= first + query
};
MEP_DEV void fill_job(const mep_diff_attn_desc& d, Job& j) {
    j.n = d.H / d.G;
    j.rows = d.Tq * j.n;
    j.len = d.Tk;
    if (d.lengths) j.len = max(0, min(j.len, G<const int>(d.lengths)[j.b]));
    j.first = d.Tk - d.Tq;
    if (d.q_start) j.first = max(-(1 << 30), min(1 << 30, G<const int>(d.q_start)[j.b]));
    if (d.causal) j.len = max(0, min(j.len, j.first + d.Tq));     // what no query sees is never read
}
MEP_DEV Job make_job(const mep_diff_attn_desc& d, int blocks, Order order, bool shared) {
    const Place p = place_of(blockIdx.x, d.B * d.G, blocks, order, shared);
    Job j;
    j.block = p.block;
    j.b = p.bg / d.G;
    j.g = p.bg - j.b * d.G;
    fill_job(d, j);
    return j;
}
// keys that any of the queries up to t may see
MEP_DEV int key_end(const mep_diff_attn_desc& d, const Job& j, int t) {
    return d.causal ? max(0, min(j.len, j.first + t + 1)) : j.len;
}

MEP_DEV bool mask_at(const mep_diff_attn_desc& d, int64_t o) {
    return d.mask_float ? G<const float>(d.mask)[o] != 0.f : G<const uint8_t>(d.mask)[o] != 0;
}
// The [B, Tk] mask's value for key k0 + lane, as it lies in memory (loaded a tile ahead of its use), and the tile's key bits:
// bit i: key k0 + i is there and not masked for every query
MEP_DEV unsigned key_raw(const mep_diff_attn_desc& d, const Job& j, int k0) {
    const int k = k0 + (int)(threadIdx.x & 63);
    if (d.mask_form != 1 || k >= j.len) return 2u;
    const int64_t o = (int64_t)j.b * d.m_sB + (int64_t)k * d.m_sK;
    return d.mask_float ? G<const uint32_t>(d.mask)[o] : (unsigned)G<const uint8_t>(d.mask)[o];
}
MEP_DEV unsigned long long key_bits(const mep_diff_attn_desc& d, const Job& j, int k0, int n, unsigned raw) {
    const int i = threadIdx.x & 63;
    return __ballot(i < n && k0 + i < j.len && (d.mask_float ? raw << 1 : raw) != 0);      // -0.0 is zero
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
    if (d.mask_form == 2) {      // all 16 at once; keys past the end read the last one's
        const int64_t o = (int64_t)j.b * d.m_sB + (int64_t)t * d.m_sQ;
        unsigned keep = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            keep |= (mask_at(d, o + (int64_t)min(k0 + 4 * h + acc_off(r), d.Tk - 1) * d.m_sK) ? 1u : 0u) << acc_off(r);
        on &= keep;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const bool ok = on >> acc_off(r) & 1;
        s1[r] = ok ? s1[r] : -INFINITY;
        s2[r] = ok ? s2[r] : -INFINITY;
    }
}

// threadIdx.x, as a value that the compiler cannot carry from one tile to the next: addresses made of it are made again (a few
// operations a tile) instead of held in registers, or worse, in scratch memory, whose loads would wait for the DMA in flight
MEP_DEV int thread_again() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// ------------------------------------------------------------------ float16: the range of the backward's operands
// float16 is exact to 2^-11 between 2^-14 and 2^16 only, and dS and P are of any size (a loss scale; the weights of many keys).  So their
// columns are multiplied by powers of two before they are rounded, and the accumulators divided by them: with
//   |dP - D| <= 2 sum|dO_t| max|v| (dq, by row),  2 max|dO_t| sum|v_k| (dk, by key),  A_1, |lam| A_2 <= w = max(1, |lam|),  |P| <= 2 w
// no value passes 2^15, and where bound and typical value are 2^6 apart (128 channels of either sign), what is 2^-19 of the
// typical value is still above 2^-24.  The maxima over a (batch row, key head) come from this kernel, a pass over the values and the
// upstream gradient: B 4, T 2048, 8 heads, 64 / 128 13 us (B 2, T 1024 7), dq 155 us and dk and dv 277, unscaled 155 and 260.  (Found
// beside the products instead, with the accumulators scaled down whenever a value passes the range: 172 and 298; at 128 / 128 437 and
// 715, with this kernel 287 and 610.)
// part p of a (batch row, key head), an n-th of its keys and of its rows: max |v|, max |dO| w, max w.  Rows that see no key are left out
// (their upstream gradient may be anything), and for dk and dv those that are too early for the keys: the last keys' gradients
// are of the size of the last rows'.
constexpr int DA_SIZE_PARTS = 64;
struct Sizes { float v, o, w; };
template <int TYPE>
struct Fit {
    static constexpr bool ON = TYPE == MEP_F16;
    // part p's first of `all` keys or rows
    static MEP_DEV int begin(int all, int p, int n) { return (int)((int64_t)all * p / n); }
    // over the keys, and the rows from `row` on
    static MEP_DEV Sizes of(uint64_t sizes, int n, const mep_diff_attn_desc& d, const Job& j, int row) {
        Sizes z = {0.f, 0.f, 1.f};
        const int p = threadIdx.x & 63;
        if (p < n) {
            const f32x4 x = G<const f32x4>(sizes)[((int64_t)j.b * d.G + j.g) * n + p];
            z.v = x[0];
            if (begin(j.rows, p + 1, n) > row) {
                z.o = x[1];
                z.w = x[2];
            }
        }
        for (int o = 32; o; o /= 2) {
            z.v = fmaxf(z.v, __shfl_xor(z.v, o));
            z.o = fmaxf(z.o, __shfl_xor(z.o, o));
            z.w = fmaxf(z.w, __shfl_xor(z.w, o));
        }
        return z;
    }
    // the n of the power of two that takes values up to `most` to under 2^15
    static MEP_DEV int lift(float most) { return max(-120, min(60, 15 - __builtin_amdgcn_frexp_expf(most))); }
};
// sum |x| over a lane's operands and its other half's
template <class M, class Op, int N>
MEP_DEV float size_sum(const Op& x) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const typename M::Frag f = x.at(i);
#pragma unroll
        for (int e = 0; e < M::E; ++e) s += fabsf((float)f[e]);
    }
    return half_sum(s);
}

template <int TYPE>
__global__ __launch_bounds__(DA_THREADS) void k_diff_sizes(mep_diff_attn_bwd_desc bd, uint64_t sizes, int parts) {
    typedef Mat<TYPE> M;
    typedef typename M::T T;
    const mep_diff_attn_desc& d = bd.f;
    __shared__ float Part[3][DA_WAVES];
    Job j;
    const int bg = blockIdx.x / parts, part = blockIdx.x - bg * parts, chunks = (d.dv + M::E - 1) / M::E;
    j.b = bg / d.G;
    j.g = bg - j.b * d.G;
    fill_job(d, j);
    auto largest = [&](const MEP_G T* p) {
        const typename M::Frag f = *reinterpret_cast<const MEP_G typename M::Frag*>(p);
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < M::E; ++e) m = fmaxf(m, fabsf((float)f[e]));
        return m;
    };
    float z[3] = {0.f, 0.f, 1.f};
    // this part's keys: those that are read; and rows
    const int k0 = Fit<TYPE>::begin(j.len, part, parts), k1 = Fit<TYPE>::begin(j.len, part + 1, parts);
    const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < (int64_t)(k1 - k0) * chunks; i += DA_THREADS) {
        const int64_t key = k0 + i / chunks;
        if (d.mask_form != 1 || mask_at(d, (int64_t)j.b * d.m_sB + key * d.m_sK)) z[0] = fmaxf(z[0], largest(vp + key * d.v_sT + i % chunks * M::E));
    }
    const int r0 = Fit<TYPE>::begin(j.rows, part, parts), r1 = Fit<TYPE>::begin(j.rows, part + 1, parts);
    const MEP_G T* op = G<const T>(bd.dout) + (int64_t)j.b * bd.o_sB + (int64_t)j.g * j.n * bd.o_sH;
    const MEP_G float* lp = G<const float>(d.lam) + (int64_t)j.b * d.lam_sB + (int64_t)j.g * j.n * d.lam_sH;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < (int64_t)(r1 - r0) * chunks; i += DA_THREADS) {
        const int row = r0 + (int)(i / chunks), t = row / j.n, head = row - t * j.n;
        if (G<const float>(d.stats)[4 * (((int64_t)j.b * d.H + j.g * j.n + head) * d.Tq + t) + 1] == 0.f) continue;      // 1 / l
        const float w = fmaxf(1.f, fabsf(lp[(int64_t)t * d.lam_sT + (int64_t)head * d.lam_sH]));
        z[1] = fmaxf(z[1], w * largest(op + (int64_t)t * bd.o_sT + (int64_t)head * bd.o_sH + i % chunks * M::E));
        z[2] = fmaxf(z[2], w);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        for (int o = 32; o; o /= 2) z[i] = fmaxf(z[i], __shfl_xor(z[i], o));
        if ((threadIdx.x & 63) == 0) Part[i][threadIdx.x >> 6] = z[i];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) z[i] = fmaxf(fmaxf(Part[i][0], Part[i][1]), fmaxf(Part[i][2], Part[i][3]));
        G<f32x4>(sizes)[blockIdx.x] = f32x4{z[0], z[1], z[2], 0.f};
    }
}

// The keys and values of a (batch, key head), tile by tile
template <int TYPE, int DK, int DV, int KT>
struct KeyTiles {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    const mep_diff_attn_desc& d;
    const MEP_G T* kp;
    const MEP_G T* vp;
    MEP_DEV KeyTiles(const mep_diff_attn_desc& desc, const Job& j) : d(desc) {
        kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH;
        vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH;
    }
    MEP_DEV void load_keys(T* tile, int k0, unsigned long long bits, int tid) const {
        const Stager<M, KT, 2 * DK> ks(tid, (unsigned)d.k_sT, [&](int c) {
            const int m = c >= DK / M::E, col = c * M::E - m * DK;
            return col < d.d ? col + (m ? (int)d.k_sM : 0) : -1;
        });
        ks.load(tile, kp + k0 * d.k_sT, (unsigned)d.k_sT, bits);
    }
    MEP_DEV void load(T* tile, int k0, unsigned long long bits) const {
        const int tid = thread_again();
        load_keys(tile, k0, bits, tid);
        const Stager<M, KT, DV> vs(tid, (unsigned)d.v_sT, [&](int c) { return c * M::E < d.dv ? c * M::E : -1; });
        vs.load(tile + KT * 2 * DK, vp + k0 * d.v_sT, (unsigned)d.v_sT, bits);
    }
};

// the rows of a wave from `first` on: lane's row, its query and head, and what the wave's keys are
struct Rows32 {
    int row0, row, t, head, wend, wfull;
    bool live;
    MEP_DEV Rows32(const mep_diff_attn_desc& d, const Job& j, int first) {
        row0 = first;
        row = row0 + (threadIdx.x & 31);
        live = row < j.rows;
        const int rr = live ? row : j.rows - 1;
        t = rr / j.n;
        head = j.g * j.n + rr - t * j.n;
        wend = row0 < j.rows ? key_end(d, j, (min(j.rows, row0 + 32) - 1) / j.n) : 0;
        wfull = d.causal ? j.first + row0 / j.n + 1 : INT_MAX;         // keys below are causal for all the wave's rows
    }
};

// A wave's accumulators (32 rows or keys x 32 N channels, transposed) times f, rounded, to rows of global memory: through LDS
// (a wave's own 32 rows of up to 128 channels), so that a row's channels are written together.  row_at(r): the row's first element, or
// null; whole: rows begin and end on 16 bytes.
template <class M, int N, class F>
MEP_DEV void write_rows(typename M::T* buf, const floatx16 (&acc)[N], float f, int n, bool whole, F row_at) {
    typedef typename M::T T;
    constexpr int P = N < 4 ? N : 4, LD = 32 * P + M::E, CH = 32 * P / M::E;
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int piece = 0; piece < N; piece += P) {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                typename VecOf<T, 4>::type v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (T)(acc[piece + i][r + e] * f);
                *reinterpret_cast<typename VecOf<T, 4>::type*>(buf + (lane & 31) * LD + 32 * i + acc_off(r) + 4 * h) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // this wave's own writes
#pragma unroll 1
        for (int i = lane; i < 32 * CH; i += 64) {
            const int r = i / CH, col = i % CH * M::E, to = 32 * piece + col;
            MEP_G T* p = row_at(r);
            if (!p || to >= n) continue;
            const typename M::Frag v = *reinterpret_cast<const typename M::Frag*>(buf + r * LD + col);
            if (whole) {
                *reinterpret_cast<MEP_G typename M::Frag*>(p + to) = v;
            } else {
#pragma unroll
                for (int e = 0; e < M::E; ++e) if (to + e < n) p[to + e] = v[e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next one is written
    }
}

// ------------------------------------------------------------------ forward
// One pass over the keys.  With e_m = 2^(s_m c - m_m) and l_m = sum e_m, out = E_1 / l_1 - lam E_2 / l_2 for E_m = sum e_m v.
// The accumulators hold X = sum round(f1 e_1 - f2 e_2) v and Y = sum round(e_2) v with f2 / f1 = rho, an estimate of
// lam l_1 / l_2 from the keys seen so far, max(f1, |f2|) = 1; at the end
//   out = X / (f1 l_1) + (f2 / (f1 l_1) - lam / l_2) Y.
// What is rounded is the difference itself, up to the estimate's error: where the maps cancel, l_1 / l_2 hardly changes along the
// keys and Y's factor vanishes.  rho is renewed, by X' = f1' (X + f2 Y) / f1 - f2' Y, at every rescaling and whenever it is
// off the sums so far (these keys' own among them) by a quarter: a few times a row, and neither operand is ever of a size
// that the row's weights do not have.  (A weight of the second map that a larger one has since replaced was rounded in both operands, and
// leaves the difference behind: up to a step of rho times its value.)
// The maxima m_m are renewed only when a score exceeds one by 8 (e <= 256: the sums are as exact), the lanes of a row agree on them, and
// the sums l_m stay lane-local to the end.
// Bound by vector operations beside the products: a step of 32 keys x 32 rows has 24 matrix instructions (64 / 128; 768 cycles) and about
// 240 others, 32 of them exponentials (1350 cycles), and two waves on a SIMD overlap them in part; s_setprio lets the wave whose products
// are ready go first (254 us -> 230).  B 2, T 4096, 8 heads, causal: 178 us; B 1, T 8192, 16 heads on 4 key heads: 466 us, 590 TFLOP/s
// of the 512 operations that a pair takes by the formula.
template <int TYPE, int DK, int DV>
struct Online {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    // The backward's e_m are to be at most 1: it gets maxima 8 up, or in float16, whose subnormals begin at 2^-14, the true ones
    static constexpr bool TOP = TYPE == MEP_F16;
    typedef Operand<M, Ge::NK, da_hold(TYPE, DK)> Q;
    Exponent<TYPE> ex;
    Q q1, q2;
    float c, lam, m1, m2, l1, l2, f1, f2, top1, top2;
    floatx16 x[DV / 32], y[DV / 32];

    MEP_DEV Online(const mep_diff_attn_desc& d, const Job& j, const Rows32& w)
        : ex(d.scale), q1(G<const T>(d.q) + (int64_t)j.b * d.q_sB + (int64_t)w.t * d.q_sT + (int64_t)w.head * d.q_sH, d.d, w.live), q2(q1.p + d.q_sM, d.d, w.live) {
        lam = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)w.t * d.lam_sT + (int64_t)w.head * d.lam_sH];
        c = ex.c;
        m1 = m2 = mul_rn(DA_MIN, c);
        l1 = l2 = f2 = 0.f;
        f1 = 1.f;
        top1 = top2 = DA_MIN;
#pragma unroll
        for (int n = 0; n < DV / 32; ++n) x[n] = y[n] = zero16();
    }
    // the 32 keys from ks on, rows r0 .. of the tile
    MEP_DEV void step(const mep_diff_attn_desc& d, const Job& j, const Rows32& w, const Reader<M, 2 * DK>& kread, const Reader<M, DV>& vread,
                      const T* kt, const T* vt, int r0, int ks, unsigned on) {
        floatx16 s1 = zero16(), s2 = zero16();
#pragma unroll
        for (int g = 0; g < Ge::NK; g += Ge::STEP)
            if (within<TYPE>(M::KS * g, d.d)) {
#pragma unroll
                for (int i = g; i < g + Ge::STEP; ++i) {
                    s1 = M::mma(kread.rows(kt, r0, i), q1.at(i), s1);
                    s2 = M::mma(kread.rows(kt, r0, Ge::NK + i), q2.at(i), s2);
                }
            }
        if (on != ~0u || ks + 32 > w.wfull || d.mask_form == 2) mask_keys(d, j, ks, on, w.t, s1, s2);
        const float a1 = max16(s1), a2 = max16(s2);
        if constexpr (TOP) {
            top1 = fmaxf(top1, a1);
            top2 = fmaxf(top2, a2);
        }
        if (__ballot(a1 * c > m1 + 8.f || a2 * c > m2 + 8.f)) {
            const float n1 = fmaxf(m1, mul_rn(half_max(a1), c)), n2 = fmaxf(m2, mul_rn(half_max(a2), c));
            const float g1 = exp2_fast(m1 - n1), g2 = exp2_fast(m2 - n2);
            l1 *= g1;
            l2 *= g2;
            m1 = n1;
            m2 = n2;
#pragma unroll
            for (int n = 0; n < DV / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[n][r] = fmaf(f2, y[n][r], x[n][r]) * g1;      // f1 E_1 alone: g2 may be 0
                    y[n][r] *= g2;
                }
            f2 = 0.f;
        }
        float u1 = 0.f, u2 = 0.f;      // sums by tiles: a long row's rounding grows with their number only
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s1[r] = ex.at(s1[r], m1);
            s2[r] = ex.at(s2[r], m2);
            u1 += s1[r];
            u2 += s2[r];
        }
        l1 += u1;
        l2 += u2;
        const float t1 = lam * half_sum(l1), t2 = half_sum(l2);
        if (__ballot(fabsf(t1 * f1 - t2 * f2) > 0.25f * fabsf(t1 * f1))) {
            const float rho = t2 > 0.f ? t1 / t2 : 0.f, h1 = 1.f / fmaxf(1.f, fabsf(rho)), h2 = rho * h1;
            const float u = h1 / f1, v = u * f2 - h2;
#pragma unroll
            for (int n = 0; n < DV / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[n][r] = fmaf(x[n][r], u, y[n][r] * v);
            f1 = h1;
            f2 = h2;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s1[r] = fmaf(s1[r], f1, -f2 * s2[r]);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < Ge::NP; ++i) {
            const Frag p = acc_frag<M>(s1, i), e = acc_frag<M>(s2, i);
#pragma unroll
            for (int n = 0; n < DV / 32; ++n)
                if (within<TYPE>(32 * n, d.dv)) {
                    const Frag v = vread.cols(vt, r0, 32 * n, i);
                    x[n] = M::mma(v, p, x[n]);
                    y[n] = M::mma(v, e, y[n]);
                }
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // the maxima that the backward gets, and 2^(m - those)
    MEP_DEV void maxima(float& n1, float& n2, float& g1, float& g2) const {      // (one rounding, as m1, m2: without keys g = 1)
        n1 = TOP ? mul_rn(half_max(top1), c) : m1 + 8.f;
        n2 = TOP ? mul_rn(half_max(top2), c) : m2 + 8.f;
        g1 = exp2_fast(m1 - n1);
        g2 = exp2_fast(m2 - n2);
    }
};

// Values wider than 128 channels (parts = 2; their accumulators would not fit beside each other) are taken by two workgroups that both
// form the scores.
// KS = 2: a workgroup takes 64 rows instead of 128, and two waves share each 32 of them, one for either half of a tile of keys; they are
// joined in LDS.  For launches of few workgroups, whose time is the chain of a row's keys while compute units stand idle (forward and dq
// at B 2, T 1024, 8 heads, 128 workgroups of 128 rows: bf16 16 / 32 35 us and 26, 39 and 32; 128 / 128 84 and 63, 77 and 59; fp32
// 64 / 128 256 and 159, 345 and 232; of 256 workgroups bf16 64 / 128 67 us and 103, but causal ones 113 and 107, 108 and 98).
template <int TYPE, int DK, int DV, int KS>
struct RowShape {
    typedef Geo<TYPE, DK, DV> Ge;
    static constexpr int RG = 4 / KS, ROWS = 32 * RG;
    static constexpr int KT = KS == 2 ? 64 : Ge::KT, KSZ = KT * 2 * DK, TSZ = KSZ + KT * DV;
    static constexpr int OUT = ROWS * (da_piece(DK > DV ? DK : DV) + Ge::M::E);      // the results pass through the tiles
    static constexpr int BUF = 2 * TSZ > OUT ? 2 * TSZ : OUT;
};
// there is a KS = 2: its tiles of 64 keys fit
constexpr bool da_two(int type, int dk, int dv) { return (type == MEP_F32 ? 4 : 2) * 2 * 64 * (2 * dk + dv) <= 160 * 1024; }

// The second waves' accumulators added to the first's: as many at a time as fit BYTES of LDS, 16 bytes of every lane side by side
template <int RG, int BYTES, int N>
MEP_DEV void join_waves(void* lds, floatx16 (&x)[N], int wave, int half) {
    constexpr int FIT = BYTES / (RG * 4096), PER = FIT < N ? FIT : N;
    static_assert(PER > 0, "LDS");
    f32x4* at = reinterpret_cast<f32x4*>(lds) + wave * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += PER) {
        if (half) {
#pragma unroll
            for (int n = n0; n < n0 + PER && n < N; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) at[((n - n0) * 4 + q) * RG * 64] = f32x4{x[n][4 * q], x[n][4 * q + 1], x[n][4 * q + 2], x[n][4 * q + 3]};
        }
        tile_sync();
        if (!half) {
#pragma unroll
            for (int n = n0; n < n0 + PER && n < N; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = at[((n - n0) * 4 + q) * RG * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][4 * q + e] += v[e];
                }
        }
        tile_sync();
    }
}

template <int TYPE, int DK, int DV, int KS>
__global__ __launch_bounds__(DA_THREADS, da_wide(TYPE, DK) || (KS == 2 && DV >= 128) ? 1 : 2) void k_diff_fwd(mep_diff_attn_desc d, int blocks, int parts) {
    typedef RowShape<TYPE, DK, DV, KS> Sh;
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    constexpr int KT = Sh::KT, RG = Sh::RG;
    __shared__ __align__(16) T Buf[Sh::BUF];      // two tiles: their keys, then their values
    __shared__ __align__(16) f32x4 Meet[KS == 2 ? 2 : 1][KS == 2 ? Sh::ROWS : 1];
    const int ld = d.dv;
    Job j = make_job(d, blocks * parts, d.causal ? LAST_LONGEST : IN_TURN, !da_wide(TYPE, DK) && KS == 1);
    if (DV == 128 && parts == 2) {
        const int c = j.block % 2 * DV;
        j.block /= 2;
        d.v += c * sizeof(T);
        d.out += c * sizeof(T);
        if (d.second) d.second += c * sizeof(T);
        if (c) d.stats = 0;
        d.dv = min(ld - c, DV);
    }
    const int h = (threadIdx.x & 63) >> 5, wave = KS == 2 ? (threadIdx.x >> 6) % RG : threadIdx.x >> 6, half = KS == 2 ? (threadIdx.x >> 6) / RG : 0;
    const Rows32 w(d, j, j.block * Sh::ROWS + wave * 32);
    const KeyTiles<TYPE, DK, DV, KT> keys(d, j);
    const Reader<M, 2 * DK> kread;
    const Reader<M, DV> vread;
    const int end = key_end(d, j, (min(j.rows, (j.block + 1) * Sh::ROWS) - 1) / j.n);

    unsigned raw = key_raw(d, j, 0);
    unsigned long long bits = key_bits(d, j, 0, KT, raw);
    if (end > 0) keys.load(Buf, 0, bits);
    raw = key_raw(d, j, KT);
    Online<TYPE, DK, DV> o(d, j, w);
    for (int k0 = 0, buf = 0; k0 < end; k0 += KT, buf ^= 1) {
        tile_sync();
        const unsigned long long now = bits;
        if (k0 + KT < end) {
            bits = key_bits(d, j, k0 + KT, KT, raw);
            keys.load(Buf + (buf ^ 1) * Sh::TSZ, k0 + KT, bits);
            raw = key_raw(d, j, k0 + 2 * KT);
        }
        const T* kt = Buf + buf * Sh::TSZ;
        int subs = KT / 32;
        if constexpr (KS == 2) asm("" : "+s"(subs));      // or the loop of one pass is folded into the outer one, whose accumulators are then copied
#pragma unroll 1
        for (int sub = half; sub < subs; sub += KS) {
            const int ks = k0 + 32 * sub;
            const unsigned on = (unsigned)(now >> (32 * sub));
            if (ks < w.wend && on) o.step(d, j, w, kread, vread, kt, kt + Sh::KSZ, 32 * sub, ks, on);
        }
    }
    o.l1 = half_sum(o.l1);
    o.l2 = half_sum(o.l2);
    float n1, n2, g1, g2;
    o.maxima(n1, n2, g1, g2);
    float l1 = o.l1 * g1, l2 = o.l2 * g2, xx, xy, yy;      // of 2^n; E_1 = xx X + xy Y, E_2 = yy Y of 2^n
    tile_sync();                             // the tiles are free
    if constexpr (KS == 2) {
        const int r = wave * 32 + (threadIdx.x & 31);
        if (h == 0) Meet[half][r] = f32x4{n1, l1, n2, l2};
        tile_sync();
        const f32x4 m = Meet[half ^ 1][r];
        const float t1 = fmaxf(n1, m[0]), t2 = fmaxf(n2, m[2]);
        const float a1 = l1 * exp2_fast(n1 - t1), b1 = m[1] * exp2_fast(m[0] - t1), a2 = l2 * exp2_fast(n2 - t2), b2 = m[3] * exp2_fast(m[2] - t2);
        l1 = a1 + b1;
        l2 = a2 + b2;
        g1 = exp2_fast(o.m1 - t1);
        g2 = exp2_fast(o.m2 - t2);
        n1 = t1;
        n2 = t2;
        xx = g1 / o.f1;
        xy = xx * o.f2;
        yy = g2;
#pragma unroll
        for (int n = 0; n < DV / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                o.x[n][i] = fmaf(o.x[n][i], xx, o.y[n][i] * xy);
                o.y[n][i] *= yy;
            }
        join_waves<RG, Sh::BUF * (int)sizeof(T)>(Buf, o.x, wave, half);
        join_waves<RG, Sh::BUF * (int)sizeof(T)>(Buf, o.y, wave, half);
        if (half) return;
        xx = yy = 1.f;
        xy = 0.f;
    } else {
        xx = g1 / o.f1;
        xy = xx * o.f2;
        yy = g2;
    }
    const float i1 = l1 > 0.f ? 1.f / l1 : l1, i2 = l2 > 0.f ? 1.f / l2 : l2;
    if (d.stats && w.live && h == 0)
        *reinterpret_cast<MEP_G f32x4*>(G<float>(d.stats) + 4 * (((int64_t)j.b * d.H + w.head) * d.Tq + w.t)) = f32x4{n1, i1, n2, i2};
    const float fx = i1 * xx, fy = i1 * xy - o.lam * i2 * yy;
    const int64_t first = (int64_t)j.b * d.Tq * d.H * ld;
    auto row_at = [&](uint64_t p, int r) -> MEP_G T* {
        const int row = w.row0 + r;
        if (row >= j.rows) return nullptr;
        const int t = row / j.n;
        return G<T>(p) + first + ((int64_t)t * d.H + j.g * j.n + row - t * j.n) * ld;
    };
    const bool whole = ld % M::E == 0;
    T* mine = Buf + wave * 32 * (da_piece(DV) + M::E);
#pragma unroll
    for (int n = 0; n < DV / 32; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o.x[n][r] = fmaf(o.x[n][r], fx, o.y[n][r] * fy);
    write_rows<M>(mine, o.x, 1.f, d.dv, whole, [&](int r) { return row_at(d.out, r); });
    if (d.second) write_rows<M>(mine, o.y, i2 * yy, d.dv, whole, [&](int r) { return row_at(d.second, r); });
}

// ------------------------------------------------------------------ forward over split keys
// Few rows against many keys (single tokens against a cache).  The tiles of keys of all (batch row, key head, 32 rows) stand in one
// row, those behind a batch row's length left out, and each of `groups` workgroups takes an equal share of it: equal work whatever
// the lengths (B 32 of up to 8192 keys, 4 key heads: 81 us, against 105 with as many tiles to a workgroup in each batch row's own
// splits), neighbouring shares on one XCD; to begin with the next rows counts as DA_SPLIT_START tiles (87 us without).  (Causal calls of
// many rows: the tiles that an item's rows do not see are dealt out too and passed over, so that a call takes as long as without the
// order of time, and less than whole: T 4096, one head, 64 / 128, bf16 80 us, 84 and 137.)  A workgroup has two waves; of a tile of 64 keys (32 where two of 64 do not fit LDS: of every other tile) a wave takes 32, and for each batch row it
// comes to it leaves its rows' maxima, sums, E_1 and E_2 in fp32; k_diff_join joins them.  Bound by reading the keys and values once,
// at 4.3 TB/s: two tiles in flight in each of two workgroups on a compute unit.
// workspace: the number of tiles before each batch row, int [B + 1]; then a part for each wave of each (workgroup, (batch row, key head,
// 32 rows)) that meet, at workgroup + (batch row, key head, 32 rows): (m1, l1, m2, l2) [R], E_1 [R][dv], E_2 [R][dv], R = min(32, rows)
constexpr int DA_SPLIT_THREADS = 128;
constexpr bool da_split_full(int type, int dk, int dv) { return dv >= 128 || dk >= 128 || type == MEP_F32; }      // all registers of a SIMD
constexpr int da_split_groups(int type, int dk, int dv) {      // that are on the chip at a time
    const int lds = (type == MEP_F32 ? 4 : 2) * 2 * da_split_keys(type, dk, dv) * (2 * dk + dv), fit = 160 * 1024 / lds, waves = da_split_full(type, dk, dv) ? 2 : 4;
    return 256 * (fit < waves ? fit : waves);
}
constexpr int64_t split_floats(int rows, int dv) { return (rows * (4 + 2 * (int64_t)dv) + 3) / 4 * 4; }
struct Parts {
    Shares all;
    int64_t stride;                    // floats of a part
    int per;                           // (key head, 32 rows) of a batch row
    gfloat* first;
};
MEP_DEV Parts parts_of(const mep_diff_attn_desc& d, int blocks, int groups, int before_end) {
    Parts p;
    p.per = d.G * blocks;
    p.all = shares_of(before_end, p.per, groups);
    p.stride = split_floats(min(32, d.Tq * (d.H / d.G)), d.dv);
    p.first = G<float>(d.workspace) + (d.B + 4) / 4 * 4;
    return p;
}

template <int TYPE, int DK, int DV>
__global__ __launch_bounds__(DA_SPLIT_THREADS, da_split_full(TYPE, DK, DV) ? 1 : 2) void k_diff_split(mep_diff_attn_desc d, int blocks, int groups) {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    constexpr int KT = da_split_keys(TYPE, DK, DV), KSZ = KT * 2 * DK, TSZ = KSZ + KT * DV;
    __shared__ __align__(16) T Buf[2 * TSZ];
    __shared__ int At[4];                        // the first wave's tiles; all; the first batch row of this share, the tiles before it
    const int tid = threadIdx.x, wave = tid >> 6, h = (tid & 63) >> 5;
    // groups is a multiple of 8
    const int self = (int)(blockIdx.x & 7) * (groups >> 3) + (int)(blockIdx.x >> 3);
    auto tiles_of = [&](int b) {
        Job r;
        r.b = b;
        fill_job(d, r);
        return r.len > 0 ? (r.len + KT - 1) / KT + DA_SPLIT_START : 0;
    };
    // the tiles before each batch row: a thread sums some rows', the threads' sums are summed up
    const int rows_each = (d.B + DA_SPLIT_THREADS - 1) / DA_SPLIT_THREADS, b0 = min(d.B, tid * rows_each), b1 = min(d.B, b0 + rows_each);
    int mine = 0;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) mine += tiles_of(b);
    int upto = mine;
    for (int o = 1; o < 64; o *= 2) {
        const int x = __shfl_up(upto, o);
        if ((tid & 63) >= o) upto += x;
    }
    if (tid == 63) {
        At[0] = upto;
        At[2] = d.B;      // (no row is looked for past the last)
    }
    __syncthreads();
    if (wave) upto += At[0];
    if (tid == DA_SPLIT_THREADS - 1) At[1] = upto;
    __syncthreads();
    const Parts parts = parts_of(d, blocks, groups, __builtin_amdgcn_readfirstlane(At[1]));
    const int64_t start = self * parts.all.share, stop = min(start + parts.all.share, parts.all.tiles);
    const bool some = start < stop;
    const int first_tile = some ? (int)(start / parts.per) : 0;      // of the batch rows' tiles
    int before = upto - mine;
    if (self == 0 || (some && before <= first_tile && first_tile < upto)) {      // (only the thread that has it looks)
        for (int b = b0; b < b1; ++b) {
            const int n = tiles_of(b);
            if (self == 0) G<int>(d.workspace)[b] = before;
            if (some && before <= first_tile && first_tile < before + n) {
                At[2] = b;
                At[3] = before;
            }
            before += n;
        }
    }
    if (self == 0 && tid == DA_SPLIT_THREADS - 1) G<int>(d.workspace)[d.B] = upto;
    if (!some) return;
    __syncthreads();

    const Reader<M, 2 * DK> kread;
    const Reader<M, DV> vread;
    int b = __builtin_amdgcn_readfirstlane(At[2]);
    before = __builtin_amdgcn_readfirstlane(At[3]);
    for (int64_t at = start; at < stop && b < d.B;) {
        const int n = __builtin_amdgcn_readfirstlane(tiles_of(b));
        const int64_t in = at - (int64_t)before * parts.per;
        if (in >= (int64_t)n * parts.per) {
            before += n;
            ++b;
            continue;
        }
        const Piece piece = piece_at(in, stop - at, n);
        const int item = piece.item;
        at += piece.taken;
        if (piece.tile0 >= piece.tile1) continue;
        Job j;
        j.b = b;
        j.g = item / blocks;
        j.block = item - j.g * blocks;
        fill_job(d, j);
        const Rows32 w(d, j, j.block * 32);
        const int begin = piece.tile0 * KT, end = min(w.wend, piece.tile1 * KT);
        const MEP_G T* kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH;
        const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH;
        auto load = [&](T* tile, int k0, unsigned long long bits) {
            const int tid = thread_again();
            const Stager<M, KT, 2 * DK, DA_SPLIT_THREADS> ks(tid, (unsigned)d.k_sT, [&](int ch) {
                const int m = ch >= DK / M::E, col = ch * M::E - m * DK;
                return col < d.d ? col + (m ? (int)d.k_sM : 0) : -1;
            });
            ks.load(tile, kp + k0 * d.k_sT, (unsigned)d.k_sT, bits);
            const Stager<M, KT, DV, DA_SPLIT_THREADS> vs(tid, (unsigned)d.v_sT, [&](int ch) { return ch * M::E < d.dv ? ch * M::E : -1; });
            vs.load(tile + KSZ, vp + k0 * d.v_sT, (unsigned)d.v_sT, bits);
        };
        unsigned raw = key_raw(d, j, begin);
        unsigned long long bits = key_bits(d, j, begin, KT, raw);
        if (begin < end) load(Buf, begin, bits);
        raw = key_raw(d, j, begin + KT);
        Online<TYPE, DK, DV> o(d, j, w);
        for (int k0 = begin, buf = 0; k0 < end; k0 += KT, buf ^= 1) {
            tile_sync();
            const unsigned long long now = bits;
            if (k0 + KT < end) {
                bits = key_bits(d, j, k0 + KT, KT, raw);
                load(Buf + (buf ^ 1) * TSZ, k0 + KT, bits);
                raw = key_raw(d, j, k0 + 2 * KT);
            }
            const int sub = KT == 64 ? wave : 0, ks = k0 + 32 * sub;      // one sub-tile a tile: the waves take turns
            const unsigned on = (unsigned)(now >> (32 * sub));
            if ((KT == 64 || ((k0 - begin) / KT & 1) == wave) && ks < end && on)
                o.step(d, j, w, kread, vread, Buf + buf * TSZ, Buf + buf * TSZ + KSZ, 32 * sub, ks, on);
        }
        tile_sync();                             // the tiles are free for the next batch row's
        float n1, n2, g1, g2;
        o.maxima(n1, n2, g1, g2);
        const float l1 = half_sum(o.l1) * g1, l2 = half_sum(o.l2) * g2;
        gfloat* part = parts.first + (part_at(self, b, parts.per, item) * 2 + wave) * parts.stride;
        const int row = tid & 31, rows = min(32, j.rows);
        if (w.live && h == 0) *reinterpret_cast<MEP_G f32x4*>(part + 4 * row) = f32x4{n1, l1, n2, l2};
        if (w.live && (l1 != 0.f || l2 != 0.f)) {      // without a key of this row here the join reads no further
            const float fx = g1 / o.f1;
            gfloat* e1 = part + 4 * rows + row * d.dv;
            gfloat* e2 = e1 + rows * d.dv;
#pragma unroll
            for (int n = 0; n < DV / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int col = 32 * n + acc_off(r) + 4 * h;
                    float a[4], b[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = fmaf(o.f2, o.y[n][r + e], o.x[n][r + e]) * fx;
                        b[e] = o.y[n][r + e] * g2;
                    }
                    if (col + 4 <= d.dv) {
                        store_f32<float, 4>(e1 + col, a);
                        store_f32<float, 4>(e2 + col, b);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (col + e < d.dv) { e1[col + e] = a[e]; e2[col + e] = b[e]; }
                    }
                }
        }
    }
}

// ------------------------------------------------------------------ backward: D and dq
// D_m = dO . (A_m v) is known beforehand only up to the roundings of the forward's out and second = A_2 v.  The error's effect on dq
// is error * sum A_m k_m, beside dS's own rounding, which comes to about r = u sqrt(sum (A_m (dP - D_m))^2) in the same units (u = 2^-9,
// in float16 2^-12).  Where the values have no mean, the error is about r (out shrinks with the keys as r does); where they have one, out
// keeps its size and the error is many times r (4096 keys, means as large as the deviations: 100 r, and dq 5 % off); and where one
// key carries the row, r itself is that error.  So the row sums of A_m dP are formed beside dS without any rounding to 16 bits, and the
// difference is put right: dq_m -= (D_m - estimate) sum A_m k_m.  At DK = 32, E_m k_m is summed beside dS (BESIDE).  Wider heads have no
// registers for that (accumulators that pass through the accumulation registers for every tile cost more than a second pass): there
// a second pass over the keys forms it where the error of a wave's 32 rows has a root mean square over 3 r, or a row rests on few
// keys (a weight over 1 / 4).  (Without a mean that is 1.3 r, 2.5 r at most in 4096 waves.  Single rows reach 8 r, and one pass
// taken twice keeps its whole launch waiting: asked of each row, B 4, T 2048, 8 heads, 64 / 128 took 185 us instead of 143.)  What the
// second pass costs where keys and values have a mean (as large as the deviation, bf16): 64 / 128 at B 2, T 4096, causal 208 -> 313 us,
// at B 4, T 2048 152 -> 229, 128 / 128 there 282 -> 474.  (In fp32 the estimate is left as it is: its error is that of the forward's
// sums over keys, 4e-7 of the terms.  Without a mean that is below dq's own; with means as large as the deviations, 2048 keys, it makes
// 9e-6 of dq, where elementary operations in 32 bits leave 2e-6.)  The sums are also lam's gradient and what dk needs.
template <int TYPE, int DK, int DV, int KS>
__global__ __launch_bounds__(DA_THREADS, DK >= 128 || (KS == 2 && DK >= 64) ? 1 : 2) void k_diff_bwd_q(mep_diff_attn_bwd_desc bd, int blocks, uint64_t sizes, int parts) {
    typedef RowShape<TYPE, DK, DV, KS> Sh;
    typedef Geo<TYPE, DK, DV> Ge;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    constexpr int KT = Sh::KT, RG = Sh::RG;
    const mep_diff_attn_desc& d = bd.f;
    __shared__ __align__(16) T Buf[Sh::BUF];      // two tiles: their keys, then their values
    __shared__ __align__(16) f32x4 Meet[KS == 2 ? 2 : 1][KS == 2 ? Sh::ROWS : 1];
    const Job j = make_job(d, blocks, d.causal ? LAST_LONGEST : IN_TURN, !da_wide(TYPE, DK) && KS == 1);
    const int h = (threadIdx.x & 63) >> 5, wave = KS == 2 ? (threadIdx.x >> 6) % RG : threadIdx.x >> 6, half = KS == 2 ? (threadIdx.x >> 6) / RG : 0;
    const Rows32 w(d, j, j.block * Sh::ROWS + wave * 32);
    const KeyTiles<TYPE, DK, DV, KT> keys(d, j);
    const Reader<M, 2 * DK> kread;
    const Reader<M, DV> vread;
    const Exponent<TYPE> ex(d.scale);
    const int end = key_end(d, j, (min(j.rows, (j.block + 1) * Sh::ROWS) - 1) / j.n);

    unsigned raw = key_raw(d, j, 0);
    unsigned long long bits = key_bits(d, j, 0, KT, raw);
    if (end > 0) keys.load(Buf, 0, bits);
    raw = key_raw(d, j, KT);
    constexpr bool HOLD = da_hold_q(TYPE, DK);
    const MEP_G T* qp = G<const T>(d.q) + (int64_t)j.b * d.q_sB + (int64_t)w.t * d.q_sT + (int64_t)w.head * d.q_sH;
    const Operand<M, Ge::NK, HOLD> q1(qp, d.d, w.live), q2(qp + d.q_sM, d.d, w.live);
    const Operand<M, Ge::NV, HOLD> g(G<const T>(bd.dout) + (int64_t)j.b * bd.o_sB + (int64_t)w.t * bd.o_sT + (int64_t)w.head * bd.o_sH, d.dv, w.live);
    float d1 = 0.f, d2 = 0.f;              // the estimates
    {
        const int64_t at = (((int64_t)j.b * d.Tq + w.t) * d.H + w.head) * d.dv;
        const MEP_G T* o = G<const T>(d.out) + at;
        const MEP_G T* o2 = G<const T>(d.second) + at;
#pragma unroll
        for (int i = 0; i < Ge::NV; ++i) {
            const int col = M::KS * i + M::E * h;
            const Frag gi = g.at(i);
            if (d.dv % M::E == 0) {
                const Frag a = row_frag<M>(o, col, d.dv, true), b = row_frag<M>(o2, col, d.dv, true);
#pragma unroll
                for (int e = 0; e < M::E; ++e) {
                    d1 = fmaf((float)gi[e], (float)a[e], d1);
                    d2 = fmaf((float)gi[e], (float)b[e], d2);
                }
            } else {
#pragma unroll
                for (int e = 0; e < M::E; ++e)
                    if (col + e < d.dv) {
                        d1 = fmaf((float)gi[e], (float)o[col + e], d1);
                        d2 = fmaf((float)gi[e], (float)o2[col + e], d2);
                    }
            }
        }
        d1 = half_sum(d1);
        d2 = half_sum(d2);
    }
    const float lam = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)w.t * d.lam_sT + (int64_t)w.head * d.lam_sH];
    d1 = fmaf(lam, d2, d1);                     // out = A_1 v - lam A_2 v
    const int64_t srow = ((int64_t)j.b * d.H + w.head) * d.Tq + w.t;
    const f32x4 st = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(d.stats) + 4 * srow);      // m1, 1 / l1, m2, 1 / l2

    constexpr bool BESIDE = TYPE != MEP_F32 && DK == 32, CORR = TYPE != MEP_F32 && DK != 32;
    float up = 1.f;                             // dS, and the estimates with it, times up (Fit)
    if constexpr (Fit<TYPE>::ON) {
        up = ldexpf(1.f, Fit<TYPE>::lift(2.f * size_sum<M, Operand<M, Ge::NV, HOLD>, Ge::NV>(g) * Fit<TYPE>::of(sizes, parts, d, j, 0).v));
        d1 *= up;
        d2 *= up;
    }
    auto above = [&](float dp, float estimate) { return Fit<TYPE>::ON ? fmaf(dp, up, -estimate) : dp - estimate; };
    float sum1 = 0.f, sum2 = 0.f, sq1 = 0.f, sq2 = 0.f, top1 = 0.f, top2 = 0.f;
    floatx16 a1[DK / 32], a2[DK / 32], b1, b2;
    b1 = b2 = zero16();
#pragma unroll
    for (int n = 0; n < DK / 32; ++n) a1[n] = a2[n] = zero16();
    int subs = KT / 32;
    if constexpr (KS == 2) asm("" : "+s"(subs));      // or the loop of one pass is folded into the outer one, whose accumulators are then copied
    for (int k0 = 0, buf = 0; k0 < end; k0 += KT, buf ^= 1) {
        tile_sync();
        const unsigned long long now = bits;
        if (k0 + KT < end) {
            bits = key_bits(d, j, k0 + KT, KT, raw);
            keys.load(Buf + (buf ^ 1) * Sh::TSZ, k0 + KT, bits);
            raw = key_raw(d, j, k0 + 2 * KT);
        }
        const T* kt = Buf + buf * Sh::TSZ;
        const T* vt = kt + Sh::KSZ;
#pragma unroll 1
        for (int sub = half; sub < subs; sub += KS) {
            const int ks = k0 + 32 * sub;
            const unsigned on = (unsigned)(now >> (32 * sub));
            if (ks >= w.wend || !on) continue;
            floatx16 s1 = zero16(), s2 = zero16(), dp = zero16();
#pragma unroll
            for (int n = 0; n < Ge::NK; n += Ge::STEP)
                if (within<TYPE>(M::KS * n, d.d)) {
#pragma unroll
                    for (int i = n; i < n + Ge::STEP; ++i) {
                        s1 = M::mma(kread.rows(kt, 32 * sub, i), q1.at(i), s1);
                        s2 = M::mma(kread.rows(kt, 32 * sub, Ge::NK + i), q2.at(i), s2);
                    }
                }
#pragma unroll
            for (int n = 0; n < Ge::NV; n += Ge::STEP)
                if (within<TYPE>(M::KS * n, d.dv)) {
#pragma unroll
                    for (int i = n; i < n + Ge::STEP; ++i) dp = M::mma(vread.rows(vt, 32 * sub, i), g.at(i), dp);
                }
            __builtin_amdgcn_s_setprio(1);
            if (on != ~0u || ks + 32 > w.wfull || d.mask_form == 2) mask_keys(d, j, ks, on, w.t, s1, s2);
            float u1 = 0.f, u2 = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {      // e_m, the row sums, and dS_m without the row's factors 1 / l1, -lam / l2
                const float e1 = ex.at(s1[r], st[0]), e2 = ex.at(s2[r], st[2]);
                u1 = fmaf(e1, dp[r], u1);
                u2 = fmaf(e2, dp[r], u2);
                if constexpr (BESIDE) {
                    s1[r] = e1;
                    s2[r] = e2;
                } else {
                    s1[r] = e1 * above(dp[r], d1);
                    s2[r] = e2 * above(dp[r], d2);
                }
                if constexpr (CORR) {
                    sq1 = fmaf(s1[r], s1[r], sq1);
                    sq2 = fmaf(s2[r], s2[r], sq2);
                    top1 = fmaxf(top1, e1);
                    top2 = fmaxf(top2, e2);
                }
            }
            sum1 += u1;
            sum2 += u2;
            Frag e1[BESIDE ? Ge::NP : 1], e2[BESIDE ? Ge::NP : 1];
            if constexpr (BESIDE) {
#pragma unroll
                for (int i = 0; i < Ge::NP; ++i) {
                    e1[i] = acc_frag<M>(s1, i);
                    e2[i] = acc_frag<M>(s2, i);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s1[r] *= above(dp[r], d1);
                    s2[r] *= above(dp[r], d2);
                }
            }
#pragma unroll
            for (int i = 0; i < Ge::NP; ++i) {
                const Frag p1 = acc_frag<M>(s1, i), p2 = acc_frag<M>(s2, i);
#pragma unroll
                for (int n = 0; n < DK / 32; ++n) {
                    if (!within<TYPE>(32 * n, d.d)) continue;
                    const Frag k1 = kread.cols(kt, 32 * sub, 32 * n, i), k2 = kread.cols(kt, 32 * sub, DK + 32 * n, i);
                    a1[n] = M::mma(k1, p1, a1[n]);
                    a2[n] = M::mma(k2, p2, a2[n]);
                    if constexpr (BESIDE) {
                        b1 = M::mma(k1, e1[i], b1);
                        b2 = M::mma(k2, e2[i], b2);
                    }
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
    }
    sum1 = half_sum(sum1);
    sum2 = half_sum(sum2);
    if constexpr (CORR) {
        sq1 = half_sum(sq1);
        sq2 = half_sum(sq2);
    }
    const bool few = CORR && w.live && fmaxf(top1 * st[1], top2 * st[3]) > 0.25f;      // (some lane has the row's largest)
    if constexpr (KS == 2) {
        const int r = wave * 32 + (threadIdx.x & 31);
        if (h == 0) Meet[half][r] = f32x4{sum1, sum2, sq1, sq2};
        __syncthreads();
        const f32x4 m = Meet[half ^ 1][r];
        sum1 += m[0];
        sum2 += m[1];
        sq1 += m[2];
        sq2 += m[3];
    }
    sum1 *= st[1];
    sum2 *= st[3];
    if (w.live && h == 0 && half == 0) {
        *reinterpret_cast<MEP_G f32x4*>(G<float>(bd.delta) + 4 * srow) = f32x4{sum1, sum2, 0.f, 0.f};
        if (bd.dlam_rows) G<float>(bd.dlam_rows)[((int64_t)j.b * d.Tq + w.t) * d.H + w.head] = -sum2;
    }
    if (!bd.dq) return;
    if constexpr (CORR) {
        constexpr float u = TYPE == MEP_F16 ? 0x1p-12f : 0x1p-9f;
        auto off = [](float error, float r) {      // (error / r)^2, finite
            const float x = error == 0.f ? 0.f : fminf(fabsf(error) / r, 1e3f);
            return x * x;
        };
        const float x = w.live ? fmaxf(off(above(-sum1, -d1), u * st[1] * sqrtf(sq1)), off(above(-sum2, -d2), u * st[3] * sqrtf(sq2))) : 0.f;
        if (__syncthreads_or(few || wave_sum(x) > 2 * 32 * 9.f)) {      // (a row is in two lanes)
            floatx16 k1[DK / 32], k2[DK / 32];
#pragma unroll
            for (int n = 0; n < DK / 32; ++n) k1[n] = k2[n] = zero16();
            for (int k0 = 0; k0 < end; k0 += KT) {      // one buffer: this pass is the rare one
                bits = key_bits(d, j, k0, KT, key_raw(d, j, k0));
                tile_sync();
                keys.load_keys(Buf, k0, bits, thread_again());
                tile_sync();
#pragma unroll 1
                for (int sub = half; sub < subs; sub += KS) {
                    const int ks = k0 + 32 * sub;
                    const unsigned on = (unsigned)(bits >> (32 * sub));
                    if (ks >= w.wend || !on) continue;
                    floatx16 s1 = zero16(), s2 = zero16();
#pragma unroll
                    for (int i = 0; i < Ge::NK; ++i) {
                        s1 = M::mma(kread.rows(Buf, 32 * sub, i), q1.at(i), s1);
                        s2 = M::mma(kread.rows(Buf, 32 * sub, Ge::NK + i), q2.at(i), s2);
                    }
                    if (on != ~0u || ks + 32 > w.wfull || d.mask_form == 2) mask_keys(d, j, ks, on, w.t, s1, s2);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        s1[r] = ex.at(s1[r], st[0]);
                        s2[r] = ex.at(s2[r], st[2]);
                    }
#pragma unroll
                    for (int i = 0; i < Ge::NP; ++i) {
                        const Frag p1 = acc_frag<M>(s1, i), p2 = acc_frag<M>(s2, i);
#pragma unroll
                        for (int n = 0; n < DK / 32; ++n) {
                            k1[n] = M::mma(kread.cols(Buf, 32 * sub, 32 * n, i), p1, k1[n]);
                            k2[n] = M::mma(kread.cols(Buf, 32 * sub, DK + 32 * n, i), p2, k2[n]);
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < DK / 32; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    a1[n][r] = fmaf(k1[n][r], above(-sum1, -d1), a1[n][r]);
                    a2[n][r] = fmaf(k2[n][r], above(-sum2, -d2), a2[n][r]);
                }
        }
    }
    if constexpr (BESIDE) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            a1[0][r] = fmaf(b1[r], above(-sum1, -d1), a1[0][r]);
            a2[0][r] = fmaf(b2[r], above(-sum2, -d2), a2[0][r]);
        }
    }
    tile_sync();                             // the tiles are free
    if constexpr (KS == 2) {
        join_waves<RG, Sh::BUF * (int)sizeof(T)>(Buf, a1, wave, half);
        join_waves<RG, Sh::BUF * (int)sizeof(T)>(Buf, a2, wave, half);
        if (half) return;
    }
    const int64_t first = (int64_t)j.b * d.Tq * d.H * 2 * d.d;
    auto row_at = [&](int m, int r) -> MEP_G T* {
        const int row = w.row0 + r;
        if (row >= j.rows) return nullptr;
        const int t = row / j.n;
        return G<T>(bd.dq) + first + (((int64_t)t * d.H + j.g * j.n + row - t * j.n) * 2 + m) * d.d;
    };
    const bool whole = d.d % M::E == 0;
    T* mine = Buf + wave * 32 * (da_piece(DK) + M::E);
    const float f = Fit<TYPE>::ON ? d.scale / up : d.scale;
    write_rows<M>(mine, a1, st[1] * f, d.d, whole, [&](int r) { return row_at(0, r); });
    write_rows<M>(mine, a2, -lam * st[3] * f, d.d, whole, [&](int r) { return row_at(1, r); });
}

// ------------------------------------------------------------------ backward: dk and dv
// A workgroup walks the rows of 32 KW keys, a wave (an accumulator column per key) those of 32.  At DK = 32 and in fp32 (one wave a
// SIMD, with all its registers) a wave forms dv and dk (ROLES = 1).  In 16 bits with wider heads the workgroup has 2 KW waves, one half
// for dv and the other for dk (ROLES = 2): both form the scores, but so neither holds more than 256 registers and two waves share a
// SIMD (in one wave, the accumulators of both pass through the accumulation registers and back for every tile: 335 us against 264
// at B 2, T 4096, 8 heads, 64 / 128, causal).  Where the blocks of keys are few, splits of the rows are summed by k_diff_kv_join.
//
// The scores lie rows x keys here, so a row's statistics are not a lane's.  They come in as a product: the accumulator starts
// at X 1 with X the row's value in three bf16 parts (24 bits) against a column of ones, one instruction for 16 registers.  With
//   s' = s - lse_m / c, lse_1 = m_1 + log2 l_1, lse_2 = m_2 + log2 l_2 - log2 |lam|:   2^(c s') = A_1, |lam| A_2
//   dP' = dP - D_1, and D_1 - D_2 added for the second map
// the rest is a product and an exponential each.  (lse_m folds a sum into the maximum, which costs last bits where the maximum is
// large: of no account in 16 bits.  In fp32, whose products take 16 times as long, the row's values are read from LDS.)
constexpr int da_roles(int type, int dk) { return dk == 32 || type == MEP_F32 ? 1 : 2; }
template <int KW, int TYPE, int DK, int DV>
struct KvShape {
    typedef Geo<TYPE, DK, DV> Ge;
    static constexpr int ROLES = da_roles(TYPE, DK), THREADS = 64 * KW * ROLES, KEYS = 32 * KW;
    static constexpr int OUT = KEYS * (da_piece(DK) + da_piece(DV) + 2 * Ge::M::E), BUF = 2 * Ge::TSZ > OUT ? 2 * Ge::TSZ : OUT;
};

typedef __bf16 bf16x8_da __attribute__((ext_vector_type(8)));
enum { X_LSE1, X_LSE2, X_D1, X_D12, X_SIGN, X_COUNT };
enum { R_M1, R_I1, R_M2, R_LI2, R_D1, R_D2, R_COUNT };

// -v, in three parts that sum to it to 24 bits, as the k = 0, 1, 2 of an operand
MEP_DEV bf16x8_da parts3(float v) {
    bf16x8_da x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (__bf16)0.f;
    v = -v;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        x[i] = (__bf16)v;
        v = sub_rn(v, (float)x[i]);
    }
    return x;
}
// the 32 rows' values x[0 .. 31], each in its row of an accumulator
MEP_DEV floatx16 row_values(const bf16x8_da* x) {
    const int lane = threadIdx.x & 63;
    bf16x8_da ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)(i < 3 && lane < 32 ? 1.f : 0.f);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[lane & 31], ones, zero16(), 0, 0, 0);
}

template <int KW, int TYPE, int DK, int DV>
__global__ __launch_bounds__(64 * KW * da_roles(TYPE, DK), da_wide(TYPE, DK) ? 1 : 2) void k_diff_bwd_kv(mep_diff_attn_bwd_desc bd, int blocks, int splits, uint64_t sizes, int parts) {
    typedef Geo<TYPE, DK, DV> Ge;
    typedef KvShape<KW, TYPE, DK, DV> Sh;
    typedef typename Ge::M M;
    typedef typename Ge::T T;
    typedef typename Ge::Frag Frag;
    constexpr int RT = Ge::KT, THREADS = Sh::THREADS, ROLES = Sh::ROLES;
    const mep_diff_attn_desc& d = bd.f;
    __shared__ __align__(16) T Buf[Sh::BUF];      // two tiles: their queries, then their upstream gradients
    constexpr bool PARTS = TYPE != MEP_F32;       // the rows' values: as products, or in fp32 as they are
    __shared__ bf16x8_da Xs[2][PARTS ? (int)X_COUNT : 1][PARTS ? RT : 1];
    __shared__ __align__(16) float Rs[2][PARTS ? 1 : (int)R_COUNT][PARTS ? 1 : RT];
    __shared__ int Ts[2][RT];                     // and queries
    __shared__ int Neg[2];                        // whether any lam of the tile is negative
    Job j = make_job(d, blocks * splits, d.causal ? FIRST_LONGEST : IN_TURN, Sh::THREADS <= 256 && !da_wide(TYPE, DK));
    const int split = j.block % splits;
    j.block /= splits;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const bool for_v = ROLES == 1 || wave < KW;
    const int key0 = j.block * Sh::KEYS + wave % KW * 32, key = key0 + (lane & 31);
    const Exponent<TYPE> ex(d.scale);
    const float c = ex.c;
    // rows that see any of the block's / the wave's keys; every one of the wave's keys: from row wfull on; the lane's key: from rmin on
    const int bstart = d.causal ? max(0, min(d.Tq, j.block * Sh::KEYS - j.first)) * j.n : 0;
    const int wstart = d.causal ? max(0, min(d.Tq, key0 - j.first)) * j.n : 0;
    const int wfull = d.causal ? max(0, min(d.Tq, key0 + 31 - j.first)) * j.n : 0;
    const int rmin = d.causal ? max(0, min(d.Tq, key - j.first)) * j.n : 0;
    // the split's share of the tiles of rows that see a key of the block
    const Range mine = split_rows(bstart / RT * RT, j.block * Sh::KEYS < j.len ? j.rows : 0, RT, split, splits);
    const int rbeg = mine.begin, rend = mine.end;

    const MEP_G T* qb = G<const T>(d.q) + (int64_t)j.b * d.q_sB + (int64_t)j.g * j.n * d.q_sH;
    const MEP_G T* ob = G<const T>(bd.dout) + (int64_t)j.b * bd.o_sB + (int64_t)j.g * j.n * bd.o_sH;
    const Reader<M, 2 * DK> qread;
    const Reader<M, DV> oread;
    auto load_rows = [&](int buf, int r0) {
        const int tid = thread_again();
        const Stager<M, RT, 2 * DK, THREADS> qs(tid, (unsigned)d.q_sT, [&](int ch) {
            const int m = ch >= DK / M::E, col = ch * M::E - m * DK;
            return col < d.d ? col + (m ? (int)d.q_sM : 0) : -1;
        });
        const Stager<M, RT, DV, THREADS> os(tid, (unsigned)bd.o_sT, [&](int ch) { return ch * M::E < d.dv ? ch * M::E : -1; });
        T* tile = Buf + buf * Ge::TSZ;
        if (j.n == 1) {
            const int left = j.rows - r0;
            const unsigned long long bits = left >= RT ? (RT == 64 ? ~0ull : 0xffffffffull) : (1ull << left) - 1;
            qs.load(tile, qb + r0 * d.q_sT, (unsigned)d.q_sT, bits);
            os.load(tile + Ge::KSZ, ob + r0 * bd.o_sT, (unsigned)bd.o_sT, bits);
        } else {      // shared heads: a tile's rows are some heads of some queries
            const int t0 = r0 / j.n, x0 = r0 - t0 * j.n;
            auto at = [&](int r, int64_t sT, int64_t sH) {
                const unsigned y = (unsigned)(x0 + r), t = y / (unsigned)j.n;
                return r0 + r < j.rows ? (int)(t * (unsigned)sT + (y - t * (unsigned)j.n) * (unsigned)sH) : -1;
            };
            qs.gather(tile, qb + t0 * d.q_sT, (unsigned)d.q_sT, [&](int r) { return at(r, d.q_sT, d.q_sH); });
            os.gather(tile + Ge::KSZ, ob + t0 * bd.o_sT, (unsigned)bd.o_sT, [&](int r) { return at(r, bd.o_sT, bd.o_sH); });
        }
    };
    // the rows' statistics on their way to LDS, a row per thread of the first wave
    f32x4 sv, dv4;
    float lv;
    int tv;
    auto fetch_stats = [&](int r0) {
        const int row = r0 + threadIdx.x;
        sv = dv4 = f32x4{0.f, 0.f, 0.f, 0.f};
        lv = 0.f;
        tv = 0;
        if (threadIdx.x < RT && row < j.rows) {
            tv = row / j.n;
            const int head = j.g * j.n + row - tv * j.n;
            const int64_t srow = ((int64_t)j.b * d.H + head) * d.Tq + tv;
            sv = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(d.stats) + 4 * srow);
            dv4 = *reinterpret_cast<const MEP_G f32x4*>(G<const float>(bd.delta) + 4 * srow);
            lv = G<const float>(d.lam)[(int64_t)j.b * d.lam_sB + (int64_t)tv * d.lam_sT + (int64_t)head * d.lam_sH];
        }
    };
    auto put_stats = [&](int buf) {
        if (threadIdx.x < 64) {
            const bool neg = __ballot(threadIdx.x < RT && lv < 0.f) != 0;
            const int i = threadIdx.x;
            if constexpr (!PARTS) {
                if (i < RT) {
                    const float v[R_COUNT] = {sv[0], sv[1], sv[2], lv * sv[3], dv4[0], dv4[1]};
#pragma unroll
                    for (int x = 0; x < R_COUNT; ++x) Rs[buf][x][i] = v[x];
                    Ts[buf][i] = tv;
                }
            } else if (i < RT) {
                // without keys, past the end (1 / l = 0) and for lam = 0: A = 0
                const float al = fabsf(lv) * sv[3];
                Xs[buf][X_LSE1][i] = parts3(sv[1] > 0.f || sv[1] != sv[1] ? (sv[0] - __log2f(sv[1])) / c : -DA_MIN);
                Xs[buf][X_LSE2][i] = parts3(al > 0.f || al != al ? (sv[2] - __log2f(al)) / c : -DA_MIN);
                Xs[buf][X_D1][i] = parts3(dv4[0]);
                Xs[buf][X_D12][i] = parts3(dv4[1] - dv4[0]);
                if (neg) Xs[buf][X_SIGN][i] = parts3(lv < 0.f ? 1.f : -1.f);
                Ts[buf][i] = tv;
            }
            if (i == 0) Neg[buf] = neg;
        }
    };
    if (rbeg < rend) {
        load_rows(0, rbeg);
        fetch_stats(rbeg);
    }
    bool on = key < j.len;
    if (on && d.mask_form == 1) on = mask_at(d, (int64_t)j.b * d.m_sB + (int64_t)key * d.m_sK);
    const int64_t krow = on ? key : 0;
    const MEP_G T* kp = G<const T>(d.k) + (int64_t)j.b * d.k_sB + (int64_t)j.g * d.k_sH + krow * d.k_sT;
    const MEP_G T* vp = G<const T>(d.v) + (int64_t)j.b * d.v_sB + (int64_t)j.g * d.v_sH + krow * d.v_sT;
    constexpr bool HOLD = da_hold(TYPE, DK);
    const Operand<M, Ge::NK, HOLD> k1(kp, d.d, on), k2(kp + d.k_sM, d.d, on);
    const bool wave_on = __ballot(on) != 0, all_on = __ballot(on) == ~0ull;
    if (rbeg < rend) put_stats(0);

    // A_1 and lam A_2 of the rows from rs on, times 2^lift
    auto maps = [&](int buf, int sub, int rs, float lift, floatx16& s1, floatx16& s2) {
        const T* qt = Buf + buf * Ge::TSZ;
        if constexpr (PARTS) {
            s1 = row_values(Xs[buf][X_LSE1] + 32 * sub);
            s2 = row_values(Xs[buf][X_LSE2] + 32 * sub);
        } else {
            s1 = s2 = zero16();
        }
#pragma unroll
        for (int n = 0; n < Ge::NK; n += Ge::STEP)
            if (within<TYPE>(M::KS * n, d.d)) {
#pragma unroll
                for (int i = n; i < n + Ge::STEP; ++i) {
                    s1 = M::mma(qread.rows(qt, 32 * sub, i), k1.at(i), s1);
                    s2 = M::mma(qread.rows(qt, 32 * sub, Ge::NK + i), k2.at(i), s2);
                }
            }
        if (!all_on || rs < wfull || d.mask_form == 2) {      // rows that see this lane's key: those from rmin on
            const int least = rmin - rs - 4 * h;
            unsigned ok = !on || least > 31 ? 0u : least > 0 ? ~0u << least : ~0u;
            if (d.mask_form == 2) {
                const int64_t o = (int64_t)j.b * d.m_sB + (int64_t)min(key, d.Tk - 1) * d.m_sK;
                unsigned keep = 0;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    keep |= (mask_at(d, o + (int64_t)Ts[buf][32 * sub + acc_off(r) + 4 * h] * d.m_sQ) ? 1u : 0u) << acc_off(r);
                ok &= keep;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s1[r] = ok >> acc_off(r) & 1 ? s1[r] : -INFINITY;
                s2[r] = ok >> acc_off(r) & 1 ? s2[r] : -INFINITY;
            }
        }
        if constexpr (PARTS) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s1[r] = exp2_fast(Fit<TYPE>::ON ? fmaf(s1[r], c, lift) : s1[r] * c);
                s2[r] = exp2_fast(Fit<TYPE>::ON ? fmaf(s2[r], c, lift) : s2[r] * c);
            }
            if (Neg[buf]) {
                const floatx16 sg = row_values(Xs[buf][X_SIGN] + 32 * sub);
#pragma unroll
                for (int r = 0; r < 16; ++r) s2[r] *= sg[r];
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int lr = 32 * sub + acc_off(r) + 4 * h;
                s1[r] = ex.at(s1[r], Rs[buf][R_M1][lr]) * Rs[buf][R_I1][lr];
                s2[r] = ex.at(s2[r], Rs[buf][R_M2][lr]) * Rs[buf][R_LI2][lr];
            }
        }
    };
    auto walk = [&](auto step) {
        for (int r0 = rbeg, buf = 0; r0 < rend; r0 += RT, buf ^= 1) {
            tile_sync();
            const bool more = r0 + RT < rend;
            if (more) {
                load_rows(buf ^ 1, r0 + RT);
                fetch_stats(r0 + RT);
            }
#pragma unroll 1
            for (int sub = 0; sub < RT / 32; ++sub) {
                const int rs = r0 + 32 * sub;
                if (wave_on && rs < j.rows && rs + 32 > wstart) step(buf, sub, rs);
            }
            if (more) put_stats(buf ^ 1);
        }
        tile_sync();                         // the tiles are free
    };
    // masked keys and keys past the lengths get zeros
    const int64_t first = (int64_t)j.b * d.Tk * d.G + j.g;
    auto key_at = [&](uint64_t p, int r, int64_t width) -> MEP_G T* {
        return key0 + r < d.Tk ? G<T>(p) + (first + (int64_t)(key0 + r) * d.G) * width : nullptr;
    };
    floatx16 av[DV / 32], a1[DK / 32], a2[DK / 32];
    auto clear_v = [&] {
#pragma unroll
        for (int n = 0; n < DV / 32; ++n) av[n] = zero16();
    };
    auto clear_k = [&] {
#pragma unroll
        for (int n = 0; n < DK / 32; ++n) a1[n] = a2[n] = zero16();
    };
    // dv += P^T dO
    auto add_v = [&](const T* ot, int sub, const floatx16& p) {
#pragma unroll
        for (int i = 0; i < Ge::NP; ++i) {
            const Frag f = acc_frag<M>(p, i);
#pragma unroll
            for (int n = 0; n < DV / 32; ++n)
                if (within<TYPE>(32 * n, d.dv)) av[n] = M::mma(oread.cols(ot, 32 * sub, 32 * n, i), f, av[n]);
        }
    };
    // dk_m += dS_m^T q_m; s1, s2: the maps
    typedef Operand<M, Ge::NV, HOLD> V;
    auto add_k = [&](const V& v, const T* qt, int buf, int sub, floatx16& s1, floatx16& s2) {
        floatx16 dp;
        if constexpr (PARTS) dp = row_values(Xs[buf][X_D1] + 32 * sub);
        else dp = zero16();
#pragma unroll
        for (int n = 0; n < Ge::NV; n += Ge::STEP)
            if (within<TYPE>(M::KS * n, d.dv)) {
#pragma unroll
                for (int i = n; i < n + Ge::STEP; ++i) dp = M::mma(oread.rows(qt + Ge::KSZ, 32 * sub, i), v.at(i), dp);
            }
        if constexpr (PARTS) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s1[r] *= dp[r];
            const floatx16 d12 = row_values(Xs[buf][X_D12] + 32 * sub);
#pragma unroll
            for (int r = 0; r < 16; ++r) s2[r] *= dp[r] + d12[r];
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int lr = 32 * sub + acc_off(r) + 4 * h;
                s1[r] *= dp[r] - Rs[buf][R_D1][lr];
                s2[r] *= dp[r] - Rs[buf][R_D2][lr];
            }
        }
#pragma unroll
        for (int i = 0; i < Ge::NP; ++i) {
            const Frag f1 = acc_frag<M>(s1, i), f2 = acc_frag<M>(s2, i);
#pragma unroll
            for (int n = 0; n < DK / 32; ++n)
                if (within<TYPE>(32 * n, d.d)) {
                    a1[n] = M::mma(qread.cols(qt, 32 * sub, 32 * n, i), f1, a1[n]);
                    a2[n] = M::mma(qread.cols(qt, 32 * sub, DK + 32 * n, i), f2, a2[n]);
                }
        }
    };
    // the powers of two that P and dS are taken to float16 with (Fit)
    int lift_v = 0, lift_k = 0;
    auto fit = [&](const V* v) {
        if constexpr (Fit<TYPE>::ON) {
            const Sizes z = Fit<TYPE>::of(sizes, parts, d, j, wstart);
            lift_v = Fit<TYPE>::lift(2.f * z.w);
            if (v) lift_k = Fit<TYPE>::lift(2.f * size_sum<M, V, Ge::NV>(*v) * z.o);
        }
    };
    // with splits, a split's sums in fp32: [splits][B, Tk, G][2 d + dv]
    auto put_part = [&](const auto& acc, int at, int n, float f) {
        if (key >= d.Tk) return;
        gfloat* p = G<float>(bd.workspace) + (((int64_t)split * d.B * d.Tk * d.G) + first + (int64_t)key * d.G) * (2 * d.d + d.dv) + at;
        constexpr int N = sizeof(acc) / sizeof(acc[0]);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = 32 * i + acc_off(r) + 4 * h;
                if (col < n) p[col] = acc[i][r] * f;
            }
    };
    auto put_v = [&](T* mine) {
        const float f = Fit<TYPE>::ON ? ldexpf(1.f, -lift_v) : 1.f;
        if (splits > 1) return put_part(av, 2 * d.d, d.dv, f);
        write_rows<M>(mine, av, f, d.dv, d.dv % M::E == 0, [&](int r) { return key_at(bd.dv, r, d.dv); });
    };
    auto put_k = [&](T* mine) {
        const float f = Fit<TYPE>::ON ? ldexpf(d.scale, -lift_k) : d.scale;
        if (splits > 1) {
            put_part(a1, 0, d.d, f);
            put_part(a2, d.d, d.d, -f);
            return;
        }
        write_rows<M>(mine, a1, f, d.d, d.d % M::E == 0, [&](int r) { return key_at(bd.dk, r, 2 * d.d); });
        write_rows<M>(mine, a2, -f, d.d, d.d % M::E == 0, [&](int r) { MEP_G T* p = key_at(bd.dk, r, 2 * d.d); return p ? p + d.d : p; });
    };
    T* vbuf = Buf + wave % KW * 32 * (da_piece(DV) + M::E);
    T* kbuf = Buf + KW * 32 * (da_piece(DV) + M::E) + wave % KW * 32 * (da_piece(DK) + M::E);
    if constexpr (ROLES == 1) {
        clear_v();
        clear_k();
        const V v(vp, d.dv, on);
        fit(&v);
        const float more = Fit<TYPE>::ON ? ldexpf(1.f, lift_k - lift_v) : 1.f;
        walk([&](int buf, int sub, int rs) {
            const T* qt = Buf + buf * Ge::TSZ;
            floatx16 s1, s2, p;
            maps(buf, sub, rs, lift_v, s1, s2);
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = s1[r] - s2[r];
            if constexpr (Fit<TYPE>::ON) {
                s1 *= more;
                s2 *= more;
            }
            add_v(qt + Ge::KSZ, sub, p);
            add_k(v, qt, buf, sub, s1, s2);
        });
        put_v(vbuf);
        put_k(kbuf);
    } else if (for_v) {
        clear_v();
        fit(nullptr);
        walk([&](int buf, int sub, int rs) {
            floatx16 s1, s2;
            maps(buf, sub, rs, lift_v, s1, s2);
#pragma unroll
            for (int r = 0; r < 16; ++r) s1[r] -= s2[r];
            add_v(Buf + buf * Ge::TSZ + Ge::KSZ, sub, s1);
        });
        put_v(vbuf);
    } else {
        clear_k();
        const V v(vp, d.dv, on);
        fit(&v);
        walk([&](int buf, int sub, int rs) {
            floatx16 s1, s2;
            maps(buf, sub, rs, lift_k, s1, s2);
            add_k(v, Buf + buf * Ge::TSZ, buf, sub, s1, s2);
        });
        put_k(kbuf);
    }
}

// ------------------------------------------------------------------ instances
// key groups of a k_diff_bwd_kv workgroup: 4 (two waves on a SIMD) where a wave's operands and accumulators fit 256 registers
constexpr int da_kw(int type, int dk) { return dk >= 128 && type != MEP_F32 ? 2 : 4; }

template <int TYPE, int DK, int DV>
void da_instance(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, uint64_t sizes, int parts) {      // splits: DA_FWD's parts, DA_SPLIT's groups
    constexpr int PV = da_piece(DV);
    if (what == DA_FWD) hipLaunchKernelGGL((k_diff_fwd<TYPE, DK, PV, 1>), dim3(grid), dim3(DA_THREADS), 0, st, d, blocks, splits);
    else if (what == DA_FWD_TWO) {
        if constexpr (da_two(TYPE, DK, PV)) hipLaunchKernelGGL((k_diff_fwd<TYPE, DK, PV, 2>), dim3(grid), dim3(DA_THREADS), 0, st, d, blocks, splits);
    } else if (what == DA_BWD_Q_TWO) {
        if constexpr (da_two(TYPE, DK, DV)) hipLaunchKernelGGL((k_diff_bwd_q<TYPE, DK, DV, 2>), dim3(grid), dim3(DA_THREADS), 0, st, *b, blocks, sizes, parts);
    }
    else if (what == DA_SPLIT) hipLaunchKernelGGL((k_diff_split<TYPE, DK, da_piece(DV)>), dim3(grid), dim3(DA_SPLIT_THREADS), 0, st, d, blocks, splits);
    else if (what == DA_BWD_Q) hipLaunchKernelGGL((k_diff_bwd_q<TYPE, DK, DV, 1>), dim3(grid), dim3(DA_THREADS), 0, st, *b, blocks, sizes, parts);
    else hipLaunchKernelGGL((k_diff_bwd_kv<da_kw(TYPE, DK), TYPE, DK, DV>), dim3(grid),
                            dim3(KvShape<da_kw(TYPE, DK), TYPE, DK, DV>::THREADS), 0, st, *b, blocks, splits, sizes, parts);
}

// the smallest instance that holds the head widths
// (its DK; its DV)
inline int da_width(int d, int dv) { return d <= 32 && dv <= 64 ? 32 : d <= 64 && dv <= 128 ? 64 : 128; }
inline int da_value_width(int d, int dv) {
    const int dk = da_width(d, dv);
    return dk == 32 ? (dv <= 32 ? 32 : 64) : dk == 64 ? (dv <= 64 ? 64 : 128) : (dv <= 128 ? 128 : 256);
}
template <int TYPE>
void da_run(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, int all, uint64_t sizes, int parts) {
    if (what == DA_SIZES) {
        if constexpr (Fit<TYPE>::ON) hipLaunchKernelGGL(k_diff_sizes<TYPE>, dim3(grid), dim3(DA_THREADS), 0, st, *b, sizes, parts);
        return;
    }
    const int dk = da_width(d.d, all), dv = da_value_width(d.d, all);      // all: the values' whole width
    if (dk == 32 && dv == 32) da_instance<TYPE, 32, 32>(what, d, b, grid, blocks, splits, st, sizes, parts);
    else if (dk == 32) da_instance<TYPE, 32, 64>(what, d, b, grid, blocks, splits, st, sizes, parts);
    else if (dk == 64 && dv == 64) da_instance<TYPE, 64, 64>(what, d, b, grid, blocks, splits, st, sizes, parts);
    else if (dk == 64) da_instance<TYPE, 64, 128>(what, d, b, grid, blocks, splits, st, sizes, parts);
    else if (dv == 128) da_instance<TYPE, 128, 128>(what, d, b, grid, blocks, splits, st, sizes, parts);
    else da_instance<TYPE, 128, 256>(what, d, b, grid, blocks, splits, st, sizes, parts);
}

void da_run_f32(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, int all, uint64_t sizes, int parts);
void da_run_bf16(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, int all, uint64_t sizes, int parts);
void da_run_f16(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, int all, uint64_t sizes, int parts);

}  // namespace mep
