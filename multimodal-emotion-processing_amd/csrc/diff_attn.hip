// mep_diff_attn_fwd / _bwd: checks, launch geometry and the join of lam's gradient (kernels: diff_attn.h).
#include <cfloat>

#include "diff_attn.h"

namespace {

using namespace mep;

// dlam[h] = -sum of A_2 dP over batch and queries, in a fixed order: a workgroup per head, threads over the rows, then the waves
constexpr int DLAM_THREADS = 1024;
__global__ __launch_bounds__(DLAM_THREADS) void k_diff_dlam(mep_diff_attn_bwd_desc bd) {
    const mep_diff_attn_desc& d = bd.f;
    __shared__ float part[DLAM_THREADS / 64];
    const int h = blockIdx.x;
    const int64_t n = (int64_t)d.B * d.Tq;
    float s = 0.f;
    auto at = [&](int64_t i) {
        const int64_t b = i / d.Tq;
        return G<const float>(bd.delta)[4 * ((b * d.H + h) * d.Tq + (i - b * d.Tq)) + 1];
    };
    int64_t i = threadIdx.x;
    for (; i + 3 * DLAM_THREADS < n; i += 4 * DLAM_THREADS) {      // four loads in flight
        const float a = at(i), b = at(i + DLAM_THREADS), c = at(i + 2 * DLAM_THREADS), e = at(i + 3 * DLAM_THREADS);
        s -= (a + b) + (c + e);
    }
    for (; i < n; i += DLAM_THREADS) s -= at(i);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = part[0];
#pragma unroll
        for (int w = 1; w < DLAM_THREADS / 64; ++w) s += part[w];
        G<float>(bd.dlam)[h] = s;
    }
}

// out = E_1 / l_1 - lam E_2 / l_2 of a row from its parts: a thread per value channel, rows side by side in a workgroup.  Bound by the
// latency of its loads: the parts' statistics are read a part a lane, and the sums of 8 parts are in flight.
__global__ __launch_bounds__(DA_THREADS) void k_diff_join(mep_diff_attn_desc d, int blocks, int groups, int per, int ld) {
    const int ch = threadIdx.x % per, lanes = min(per, 64), lane = threadIdx.x % lanes;
    const int64_t all = (int64_t)d.B * d.Tq * d.H, at = (int64_t)blockIdx.x * (DA_THREADS / per) + threadIdx.x / per;
    const int64_t r = min(at, all - 1);      // (b, t, head); lanes without a row work on the last one and write nothing
    const int64_t bt = r / d.H;
    const int head = (int)(r - bt * d.H), b = (int)(bt / d.Tq), t = (int)(bt - (int64_t)b * d.Tq);
    const int n = d.H / d.G, g = head / n, row = t * n + head - g * n, rows = min(32, d.Tq * n);
    const int* before = reinterpret_cast<const int*>(d.workspace);
    const Parts ps = parts_of(d, blocks, groups, before[d.B]);
    // the row's tiles are tile .. tile + tiles - 1 of all
    const int item = g * blocks + row / 32, tiles = before[b + 1] - before[b];
    const Meet meet = meet_of((int64_t)before[b] * ps.per + (int64_t)item * tiles, tiles, ps.all.share);
    const int parts = 2 * meet.count;
    const int64_t stride = ps.stride;
    const gfloat* part = ps.first + part_at(meet.first, b, ps.per, item) * 2 * stride;
    const int lr = row & 31;
    auto stats = [&](int p) { return *reinterpret_cast<const MEP_G f32x4*>(part + p * stride + 4 * lr); };
    float m1 = -FLT_MAX, m2 = -FLT_MAX;      // (without keys the backward gets finite ones)
    for (int p = lane; p < parts; p += lanes) {
        const f32x4 s = stats(p);
        m1 = fmaxf(m1, s[0]);
        m2 = fmaxf(m2, s[2]);
    }
    for (int o = lanes / 2; o; o /= 2) {
        m1 = fmaxf(m1, __shfl_xor(m1, o));
        m2 = fmaxf(m2, __shfl_xor(m2, o));
    }
    float l1 = 0.f, l2 = 0.f, e1 = 0.f, e2 = 0.f;
    const gfloat* v1 = part + 4 * rows + lr * d.dv + min(ch, d.dv - 1);
    const gfloat* v2 = v1 + rows * d.dv;
    for (int p0 = 0; p0 < parts; p0 += lanes) {
        float w1 = 0.f, w2 = 0.f;
        bool on = false;                          // without a key of this row there, no sums are written
        if (p0 + lane < parts) {
            const f32x4 s = stats(p0 + lane);
            on = s[1] != 0.f || s[3] != 0.f;
            w1 = on ? exp2_fast(s[0] - m1) : 0.f;
            w2 = on ? exp2_fast(s[2] - m2) : 0.f;
            l1 = on ? fmaf(s[1], w1, l1) : l1;
            l2 = on ? fmaf(s[3], w2, l2) : l2;
        }
        const int count = min(lanes, parts - p0);
        for (int i = 0; i < count; i += 8) {
            float a[8], c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t o = min(p0 + i + j, parts - 1) * stride;
                a[j] = v1[o];
                c[j] = v2[o];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {         // (i + j < lanes, a multiple of 8; weights behind the last part are not on)
                const float u1 = __shfl(w1, i + j, lanes), u2 = __shfl(w2, i + j, lanes);
                const bool x = __shfl((int)on, i + j, lanes);
                e1 = x ? fmaf(a[j], u1, e1) : e1;
                e2 = x ? fmaf(c[j], u2, e2) : e2;
            }
        }
    }
    for (int o = lanes / 2; o; o /= 2) {
        l1 += __shfl_xor(l1, o);
        l2 += __shfl_xor(l2, o);
    }
    if (at >= all) return;
    const float i1 = l1 > 0.f ? 1.f / l1 : l1, i2 = l2 > 0.f ? 1.f / l2 : l2;
    const float lam = G<const float>(d.lam)[(int64_t)b * d.lam_sB + (int64_t)t * d.lam_sT + (int64_t)head * d.lam_sH];
    if (d.stats && ch == 0) *reinterpret_cast<MEP_G f32x4*>(G<float>(d.stats) + 4 * (((int64_t)b * d.H + head) * d.Tq + t)) = f32x4{m1, i1, m2, i2};
    if (ch >= d.dv) return;
    auto put = [&](uint64_t p, float v) {
        const int64_t o = r * ld + ch;
        if (d.type == MEP_F32) G<float>(p)[o] = v;
        else if (d.type == MEP_BF16) G<__bf16>(p)[o] = (__bf16)v;
        else G<_Float16>(p)[o] = (_Float16)v;
    };
    put(d.out, fmaf(e1, i1, -lam * (e2 * i2)));
    if (d.second) put(d.second, e2 * i2);
}

// rows that can be read 16 bytes at a time, a tile of 64 time steps with all its heads and maps within 2 GiB (the DMA's 32-bit
// byte offsets)
bool rows_ok(const mep_diff_attn_desc& d, uint64_t p, int64_t sB, int64_t sT, int64_t sH, int64_t sM, bool heads) {
    const int64_t V = d.type == MEP_F32 ? 4 : 8, h = heads ? d.H / d.G : 0;
    return p % 16 == 0 && sB % V == 0 && sT % V == 0 && sH % V == 0 && sM % V == 0 && sT >= 0 && sT < 1 << 23 && sM >= 0 && sM < 1 << 28 &&
           (!heads || (sH >= 0 && sH * h < 1 << 28)) && 64 * sT + sM + sH * h < (V << 27) - 512;
}
bool keys_ok(const mep_diff_attn_desc& d) {
    return rows_ok(d, d.k, d.k_sB, d.k_sT, d.k_sH, d.k_sM, false) && rows_ok(d, d.v, d.v_sB, d.v_sT, d.v_sH, 0, false);
}
bool inputs_ok(const mep_diff_attn_desc& d) { return rows_ok(d, d.q, d.q_sB, d.q_sT, d.q_sH, d.q_sM, true) && keys_ok(d); }

// the workgroups of a launch over `items` rows or keys per (batch, key head), `per` each, or -1 (too many)
int64_t plan(const mep_diff_attn_desc& d, int64_t items, int per, int& blocks) {
    blocks = (int)((items + per - 1) / per);
    const int64_t grid = (int64_t)blocks * d.B * d.G;
    return grid < 1 << 23 ? grid : -1;            // of up to 512 threads: 2^32 threads are a launch's most
}

// dk and dv from the splits' sums, in order
template <class T>
__global__ __launch_bounds__(DA_THREADS) void k_diff_kv_join(mep_diff_attn_bwd_desc bd, int splits) {
    const mep_diff_attn_desc& d = bd.f;
    const int w = 2 * d.d + d.dv;
    const int64_t n = (int64_t)d.B * d.Tk * d.G, total = n * w;
    for (int64_t i = (int64_t)blockIdx.x * DA_THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * DA_THREADS) {
        const gfloat* p = G<const float>(bd.workspace) + i;
        float s = p[0];
        for (int k = 1; k < splits; ++k) s += p[k * total];
        const int64_t row = i / w;
        const int c = (int)(i - row * w);
        if (c < 2 * d.d) G<T>(bd.dk)[row * 2 * d.d + c] = (T)s;
        else G<T>(bd.dv)[row * d.dv + c - 2 * d.d] = (T)s;
    }
}

// Whether the keys of a forward are split (groups > 0), and over how many workgroups.  Worth it where the rows are few: up to 32 a
// (batch row, key head) leave three of k_diff_fwd's four waves idle (with 4 key heads, 64 / 128, full and ragged caches: 64 batch rows of
// 8192 keys 336 and 330 us whole, 213 and 120 split; 64 of 1024 49 and 48, 48 and 39; 128 of 1024 55 and 52, 66 and 54; 64 of 512
// 30 and 28, 37 and 30), and more rows too when they make up to 32 workgroups and there are 1024 keys (32 workgroups against
// 4096 keys: bf16 16 / 32 79 us whole, 37 split, 64 / 128 141 and 82; 56 against 2048: 128 / 128 98 and 145).  As many workgroups
// as are on the chip at a time, and 4 tiles for each.
struct Split { int blocks, groups; };
Split split_of(const mep_diff_attn_desc& d) {
    Split s = {0, 0};
    const int64_t rows = (int64_t)d.Tq * (d.H / d.G), pairs = (int64_t)d.B * d.G;
    const bool few = rows <= 32 && d.Tk >= (pairs < 512 ? 1024 : 2048), none = rows > 32 && d.Tk >= 1024 && pairs * ((rows + DA_ROWS - 1) / DA_ROWS) <= 32;
    if (pairs == 0 || rows == 0 || !(few || none)) return s;
    s.blocks = (int)((rows + 31) / 32);
    const int dk = da_width(d.d, d.dv), dv = da_piece(da_value_width(d.d, d.dv)), kt = da_split_keys(d.type, dk, dv);
    const int64_t items = pairs * s.blocks, all = (d.Tk + kt - 1) / kt, want = (items * all + 3) / 4, most = da_split_groups(d.type, dk, dv);
    if (items >= 1 << 20 || d.B * (all + DA_SPLIT_START) >= INT_MAX) return s;      // there are enough rows, or too many tiles to count in 32 bits
    s.groups = (int)((want < most ? want : most) + 7) / 8 * 8;
    return s;
}
int64_t split_bytes(const mep_diff_attn_desc& d, const Split& s) {
    const int64_t rows = (int64_t)d.Tq * (d.H / d.G), parts = s.groups + (int64_t)d.B * d.G * s.blocks;
    return ((d.B + 4) / 4 * 4 + parts * 2 * split_floats((int)(rows < 32 ? rows : 32), da_piece(d.dv))) * 4;
}

void run(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, int64_t grid, int blocks, int splits, hipStream_t st, int dv, uint64_t sizes = 0, int parts = 0) {
    if (d.type == MEP_F32) da_run_f32(what, d, b, (unsigned)grid, blocks, splits, st, dv, sizes, parts);
    else if (d.type == MEP_BF16) da_run_bf16(what, d, b, (unsigned)grid, blocks, splits, st, dv, sizes, parts);
    else da_run_f16(what, d, b, (unsigned)grid, blocks, splits, st, dv, sizes, parts);
}

// Into how many workgroups the rows of a block of keys are split: until there are two for every compute unit, 4 tiles of rows each at
// least, 8 at most (each leaves its sums in fp32, which k_diff_kv_join adds: 10 us at B 2, T 1024, 4 key heads, 64 / 64, where dk and dv
// take 187 us in fp32 split and 480 whole)
int kv_splits(const mep_diff_attn_desc& d) {
    const int dk = da_width(d.d, d.dv), per = 32 * da_kw(d.type, dk), tile = d.type == MEP_F32 ? 32 : 64;
    const int64_t grid = (int64_t)d.B * d.G * ((d.Tk + per - 1) / per), tiles = ((int64_t)d.Tq * (d.H / d.G) + tile - 1) / tile;
    if (grid == 0) return 1;
    int64_t n = 512 / grid;
    n = n > tiles / 4 ? tiles / 4 : n;
    return (int)(n < 1 ? 1 : n > 8 ? 8 : n);
}

// bytes of the splits' sums, and behind them of k_diff_sizes' parts: 32 keys or rows each, DA_SIZE_PARTS at most (a lane's worth)
int64_t kv_bytes(const mep_diff_attn_desc& d) {
    const int n = kv_splits(d);
    return n > 1 ? ((int64_t)n * d.B * d.Tk * d.G * (2 * d.d + d.dv) * 4 + 15) / 16 * 16 : 0;
}
int size_parts(const mep_diff_attn_desc& d) {
    const int64_t rows = (int64_t)d.Tq * (d.H / d.G), pairs = (int64_t)d.B * d.G;
    if (d.type != MEP_F16 || pairs == 0) return 0;
    int64_t n = ((rows > d.Tk ? rows : d.Tk) + 31) / 32;
    n = n > DA_SIZE_PARTS ? DA_SIZE_PARTS : n;
    if (n * pairs >= 1 << 23) n = ((1 << 23) - 1) / pairs;
    return (int)(n < 1 ? 1 : n);
}

// Whether two waves share a row's keys (KS = 2) in a launch of `grid` workgroups of 128 rows, over dv channels of the values at a time:
// while that leaves half of the compute units idle; causal ones, of which the longest are left at the end, while there is one for each
bool two_waves(const mep_diff_attn_desc& d, int64_t grid, int dv) {
    const int dk = da_width(d.d, d.dv), width = da_value_width(d.d, d.dv);
    return grid <= (d.causal ? 256 : 128) && d.Tk > 64 && da_two(d.type, dk, width < dv ? width : dv);
}

bool attn_shape_ok(const mep_diff_attn_desc& d) {
    if (d.B < 0 || d.Tq < 0 || d.Tk < 0 || d.H < 1 || d.G < 1 || d.H % d.G || d.type < MEP_F32 || d.type > MEP_F16) return false;
    if (d.d < 1 || d.d > MEP_DIFF_ATTN_MAX_D || d.dv < 1 || d.dv > MEP_DIFF_ATTN_MAX_DV) return false;
    if (d.Tk >= 1 << 30 || (int64_t)d.Tq * (d.H / d.G) >= 1 << 30 || (int64_t)d.B * d.G >= 1 << 30) return false;
    return true;
}
bool attn_ok(const mep_diff_attn_desc& d) {
    if (!attn_shape_ok(d)) return false;
    if (!(d.scale > 0.f && d.scale <= 1e6f) || d.mask_form < 0 || d.mask_form > 2 || (d.mask_form != 0) != (d.mask != 0)) return false;
    const bool empty = d.B == 0 || d.Tq == 0;
    return empty || (d.q && d.lam && d.out && (d.Tk == 0 || (d.k && d.v)));
}

// 16 bytes of a packed row per thread
template <class T>
__global__ __launch_bounds__(DA_THREADS) void k_pack_rows(mep_pack_rows_desc d, int chunks, int64_t total) {
    constexpr int E = 16 / (int)sizeof(T);
    for (int64_t i = (int64_t)blockIdx.x * DA_THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * DA_THREADS) {
        const int64_t row = i / chunks;
        const int col = (int)(i - row * chunks) * E;
        int64_t r = row;
        const int m = (int)(r % d.M);
        r /= d.M;
        const int h = (int)(r % d.H);
        r /= d.H;
        const int64_t t = r % d.T, b = r / d.T;
        const MEP_G T* src = G<const T>(d.x) + b * d.sB + t * d.sT + h * d.sH + m * d.sM;
        typename VecOf<T, E>::type v;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = col + e < d.n ? src[(int64_t)(col + e) * d.sN] : (T)0.f;
        *reinterpret_cast<MEP_G typename VecOf<T, E>::type*>(G<T>(d.y) + row * chunks * E + col) = v;
    }
}

}  // namespace

extern "C" int mep_pack_rows(const mep_pack_rows_desc* desc, mep_stream_t stream) {
    if (!desc || desc->B < 0 || desc->T < 0 || desc->H < 1 || desc->M < 1 || desc->n < 1 || desc->type < MEP_F32 || desc->type > MEP_F16 ||
        !desc->x || !desc->y || desc->y % 16) {
        mep_set_error("mep_pack_rows: invalid descriptor");
        return MEP_EINVAL;
    }
    const int E = desc->type == MEP_F32 ? 4 : 8, chunks = (desc->n + E - 1) / E;
    const int64_t total = (int64_t)desc->B * desc->T * desc->H * desc->M * chunks, want = (total + DA_THREADS - 1) / DA_THREADS;
    if (total == 0) return 0;
    const dim3 grid((unsigned)(want < 8192 ? want : 8192)), block(DA_THREADS);
    if (desc->type == MEP_F32) hipLaunchKernelGGL(k_pack_rows<float>, grid, block, 0, (hipStream_t)stream, *desc, chunks, total);
    else if (desc->type == MEP_BF16) hipLaunchKernelGGL(k_pack_rows<__bf16>, grid, block, 0, (hipStream_t)stream, *desc, chunks, total);
    else hipLaunchKernelGGL(k_pack_rows<_Float16>, grid, block, 0, (hipStream_t)stream, *desc, chunks, total);
    return mep_check_launch("mep_pack_rows");
}

extern "C" int mep_diff_attn_fwd(const mep_diff_attn_desc* desc, mep_stream_t stream) {
    if (!desc || !attn_ok(*desc) || !desc->stats != !desc->second) {
        mep_set_error("mep_diff_attn_fwd: invalid descriptor");
        return MEP_EINVAL;
    }
    const mep_diff_attn_desc& d = *desc;
    if (d.B == 0 || d.Tq == 0) return 0;
    if (!inputs_ok(d)) { mep_set_error("mep_diff_attn_fwd: rows that cannot be read 16 bytes at a time"); return MEP_EINVAL; }
    int blocks;
    int64_t grid = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS, blocks);
    if (grid < 0) { mep_set_error("mep_diff_attn_fwd: too many rows for one launch"); return MEP_EINVAL; }
    hipStream_t st = (hipStream_t)stream;
    const Split s = split_of(d);
    const int es = d.type == MEP_F32 ? 4 : 2, half = da_piece(d.dv);
    if (!s.groups || !d.workspace) {
        const int parts = d.dv > half ? 2 : 1;
        const bool two = two_waves(d, grid * parts, 128);
        if (two) grid = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS / 2, blocks);
        if (grid * parts >= 1 << 23) { mep_set_error("mep_diff_attn_fwd: too many rows for one launch"); return MEP_EINVAL; }
        run(two ? DA_FWD_TWO : DA_FWD, d, nullptr, grid * parts, blocks, parts, st, d.dv);
        return mep_check_launch("mep_diff_attn_fwd");
    }
    // values of more than 128 channels in two launches: their accumulators would not fit beside each other
    for (int c = 0; c < d.dv; c += half) {
        mep_diff_attn_desc p = d;
        p.dv = d.dv - c < half ? d.dv - c : half;
        p.v += (uint64_t)c * es;
        p.out += (uint64_t)c * es;
        if (p.second) p.second += (uint64_t)c * es;
        if (c) p.stats = 0;
        run(DA_SPLIT, p, nullptr, s.groups, s.blocks, s.groups, st, d.dv);
        int per = 32;
        while (per < p.dv) per *= 2;
        const int64_t rows = (int64_t)d.B * d.Tq * d.H, side = DA_THREADS / per;
        hipLaunchKernelGGL(k_diff_join, dim3((unsigned)((rows + side - 1) / side)), dim3(DA_THREADS), 0, st, p, s.blocks, s.groups, per, d.dv);
        const int rc = mep_check_launch("mep_diff_attn_fwd");
        if (rc) return rc;
    }
    return 0;
}

extern "C" int64_t mep_diff_attn_bwd_workspace(const mep_diff_attn_desc* desc) {
    if (!desc || !attn_shape_ok(*desc)) { mep_set_error("mep_diff_attn_bwd_workspace: invalid descriptor"); return MEP_EINVAL; }
    return kv_bytes(*desc) + (int64_t)size_parts(*desc) * desc->B * desc->G * 16;
}

extern "C" int64_t mep_diff_attn_workspace(const mep_diff_attn_desc* desc) {
    if (!desc || !attn_shape_ok(*desc)) { mep_set_error("mep_diff_attn_workspace: invalid descriptor"); return MEP_EINVAL; }
    const Split s = split_of(*desc);
    return s.groups ? split_bytes(*desc, s) : 0;
}

extern "C" int mep_diff_attn_bwd(const mep_diff_attn_bwd_desc* desc, mep_stream_t stream) {
    if (!desc || !attn_ok(desc->f)) { mep_set_error("mep_diff_attn_bwd: invalid descriptor"); return MEP_EINVAL; }
    const mep_diff_attn_bwd_desc& b = *desc;
    const mep_diff_attn_desc& d = b.f;
    const bool rows = d.B > 0 && d.Tq > 0, keys = d.B > 0 && d.Tk > 0;
    if ((rows && (!d.stats || !d.second || !b.dout || !b.delta)) || (keys && (!b.dk != !b.dv || !d.k || !d.v))) {
        mep_set_error("mep_diff_attn_bwd: a missing operand");
        return MEP_EINVAL;
    }
    if ((rows && (!inputs_ok(d) || !rows_ok(d, b.dout, b.o_sB, b.o_sT, b.o_sH, 0, true))) || (keys && !keys_ok(d))) {
        mep_set_error("mep_diff_attn_bwd: rows that cannot be read 16 bytes at a time");
        return MEP_EINVAL;
    }
    const int parts = rows || keys ? size_parts(d) : 0;
    if (parts && (!b.workspace || b.workspace % 16)) {
        mep_set_error("mep_diff_attn_bwd: float16 without a workspace");
        return MEP_EINVAL;
    }
    hipStream_t st = (hipStream_t)stream;
    int qb, kb;
    const int64_t kg = plan(d, d.Tk, 32 * da_kw(d.type, da_width(d.d, d.dv)), kb);
    int64_t qg = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS, qb);
    if (qg < 0 || kg < 0) { mep_set_error("mep_diff_attn_bwd: too many rows for one launch"); return MEP_EINVAL; }
    const uint64_t sizes = b.workspace + (uint64_t)kv_bytes(d);
    if (parts) run(DA_SIZES, d, &b, (int64_t)d.B * d.G * parts, 0, 1, st, d.dv, sizes, parts);
    if (rows) {
        const bool two = two_waves(d, qg, 256);
        if (two) qg = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS / 2, qb);
        run(two ? DA_BWD_Q_TWO : DA_BWD_Q, d, &b, qg, qb, 1, st, d.dv, sizes, parts);
    }
    if (keys && b.dk) {
        const int splits = b.workspace ? kv_splits(d) : 1;
        run(DA_BWD_KV, d, &b, kg * splits, kb, splits, st, d.dv, sizes, parts);
        if (splits > 1) {
            const int64_t want = ((int64_t)d.B * d.Tk * d.G * (2 * d.d + d.dv) + DA_THREADS - 1) / DA_THREADS;
            const dim3 grid((unsigned)(want < 4096 ? want : 4096)), block(DA_THREADS);
            if (d.type == MEP_F32) hipLaunchKernelGGL(k_diff_kv_join<float>, grid, block, 0, st, b, splits);
            else if (d.type == MEP_BF16) hipLaunchKernelGGL(k_diff_kv_join<__bf16>, grid, block, 0, st, b, splits);
            else hipLaunchKernelGGL(k_diff_kv_join<_Float16>, grid, block, 0, st, b, splits);
        }
    }
    if (b.dlam) hipLaunchKernelGGL(k_diff_dlam, dim3(d.H), dim3(DLAM_THREADS), 0, st, b);
    return mep_check_launch("mep_diff_attn_bwd");
}
