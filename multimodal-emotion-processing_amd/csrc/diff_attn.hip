// mep_diff_attn_fwd / _bwd: checks, launch geometry and the join of lam's gradient (kernels: diff_attn.h).
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

// rows that can be read 16 bytes at a time, a tile of 64 time steps with all its heads and maps within 2^30 elements (the DMA's
// 32-bit byte offsets)
bool rows_ok(const mep_diff_attn_desc& d, uint64_t p, int64_t sB, int64_t sT, int64_t sH, int64_t sM, bool heads) {
    const int64_t V = d.type == MEP_F32 ? 4 : 8;
    return p % 16 == 0 && sB % V == 0 && sT % V == 0 && sH % V == 0 && sM % V == 0 && sT >= 0 && sT < 1 << 23 && sM >= 0 && sM < 1 << 28 &&
           (!heads || (sH >= 0 && sH * (d.H / d.G) < 1 << 28));
}
bool inputs_ok(const mep_diff_attn_desc& d) {
    return rows_ok(d, d.q, d.q_sB, d.q_sT, d.q_sH, d.q_sM, true) && rows_ok(d, d.k, d.k_sB, d.k_sT, d.k_sH, d.k_sM, false) &&
           rows_ok(d, d.v, d.v_sB, d.v_sT, d.v_sH, 0, false);
}

// the workgroups of a launch over `items` rows or keys per (batch, key head), `per` each, or -1 (too many)
int64_t plan(const mep_diff_attn_desc& d, int64_t items, int per, int& blocks) {
    blocks = (int)((items + per - 1) / per);
    const int64_t grid = (int64_t)blocks * d.B * d.G;
    return grid < 1 << 23 ? grid : -1;            // of up to 512 threads: 2^32 threads are a launch's most
}

void run(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, int64_t grid, int blocks, hipStream_t st) {
    if (d.type == MEP_F32) da_run_f32(what, d, b, (unsigned)grid, blocks, st);
    else if (d.type == MEP_BF16) da_run_bf16(what, d, b, (unsigned)grid, blocks, st);
    else da_run_f16(what, d, b, (unsigned)grid, blocks, st);
}

bool attn_ok(const mep_diff_attn_desc& d) {
    if (d.B < 0 || d.Tq < 0 || d.Tk < 0 || d.H < 1 || d.G < 1 || d.H % d.G || d.type < MEP_F32 || d.type > MEP_F16) return false;
    if (d.d < 1 || d.d > MEP_DIFF_ATTN_MAX_D || d.dv < 1 || d.dv > MEP_DIFF_ATTN_MAX_DV) return false;
    if (d.Tk >= 1 << 30 || (int64_t)d.Tq * (d.H / d.G) >= 1 << 30 || (int64_t)d.B * d.G >= 1 << 30) return false;
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
    const int64_t grid = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS, blocks);
    if (grid < 0) { mep_set_error("mep_diff_attn_fwd: too many rows for one launch"); return MEP_EINVAL; }
    run(DA_FWD, d, nullptr, grid, blocks, (hipStream_t)stream);
    return mep_check_launch("mep_diff_attn_fwd");
}

extern "C" int mep_diff_attn_bwd(const mep_diff_attn_bwd_desc* desc, mep_stream_t stream) {
    if (!desc || !attn_ok(desc->f)) { mep_set_error("mep_diff_attn_bwd: invalid descriptor"); return MEP_EINVAL; }
    const mep_diff_attn_bwd_desc& b = *desc;
    const mep_diff_attn_desc& d = b.f;
    const bool rows = d.B > 0 && d.Tq > 0, keys = d.B > 0 && d.Tk > 0;
    if ((rows && (!d.stats || !d.second || !b.dout || !b.delta)) || (keys && (!b.dk != !b.dv))) {
        mep_set_error("mep_diff_attn_bwd: a missing operand");
        return MEP_EINVAL;
    }
    if (rows && (!inputs_ok(d) || !rows_ok(d, b.dout, b.o_sB, b.o_sT, b.o_sH, 0, true))) {
        mep_set_error("mep_diff_attn_bwd: rows that cannot be read 16 bytes at a time");
        return MEP_EINVAL;
    }
    hipStream_t st = (hipStream_t)stream;
    int qb, kb;
    const int64_t qg = plan(d, (int64_t)d.Tq * (d.H / d.G), DA_ROWS, qb),
                  kg = plan(d, d.Tk, 32 * da_kw(d.type, da_width(d.d, d.dv)), kb);
    if (qg < 0 || kg < 0) { mep_set_error("mep_diff_attn_bwd: too many rows for one launch"); return MEP_EINVAL; }
    if (rows) run(DA_BWD_Q, d, &b, qg, qb, st);
    if (keys && b.dk) run(DA_BWD_KV, d, &b, kg, kb, st);
    if (b.dlam) hipLaunchKernelGGL(k_diff_dlam, dim3(d.H), dim3(DLAM_THREADS), 0, st, b);
    return mep_check_launch("mep_diff_attn_bwd");
}
