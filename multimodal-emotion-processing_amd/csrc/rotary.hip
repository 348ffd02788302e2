// mep_rotary: rotary positions.  Pair i of a head's first `rot` channels is turned by the angle
// a = pos * freqs[i]:  y1 = A (x1 cos a - x2 sin a),  y2 = A (x2 cos a + x1 sin a);  the channels
// behind `rot` are copied.  The pairs are channels (i, i + rot / 2), or (2i, 2i + 1) interleaved.
// The gradient is the same turn by -a (`inverse`).
//
// The angle is taken in 64 bits and reduced to the nearest quarter turn there: in 32 bits a
// position of 10^5 has lost 2^-7 turns before its cosine is formed.  What is left, within an eighth of
// a turn, goes to 32 bits and through the Taylor series of sine and cosine.
//
// Bound by memory: 2 D elements per head and token against ~20 operations per pair and token.  A thread
// owns one 2V-channel item of one token (V pairs, or 2V copied channels), forms its V sines once and walks
// the heads with them; the heads are split over threads only where tokens alone do not fill the chip.
// 4 x 8192 tokens of 16 + 4 heads of 128 in bf16: 73 us, 4.6 TB/s.
#include "elem.h"

namespace {

using namespace mep;

// sin / cos of 2 pi x, x in [-1/8, 1/8]: Taylor to x^9 and x^10 (the next terms are below 2e-9 and 1e-10)
MEP_DEV void sincos_turns(float x, float& s, float& c) {
    const float t = x * 6.283185307179586f, t2 = t * t;
    s = fmaf(t * t2, fmaf(t2, fmaf(t2, fmaf(t2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), t);
    c = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
}

constexpr int ROT_THREADS = 256;

template <int TYPE, int V, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void k_rotary(mep_rotary_desc d, int np, int ni, int hsplit) {
    typedef typename ElemOf<TYPE>::T T;
    const int64_t id = (int64_t)blockIdx.x * ROT_THREADS + threadIdx.x;
    const int64_t unit = id / ni;
    const int item = (int)(id - unit * ni);
    const int64_t tok = unit / hsplit;
    const int hs = (int)(unit - tok * hsplit);
    if (tok >= (int64_t)d.B * d.T) return;
    const int b = (int)(tok / d.T), t = (int)(tok - (int64_t)b * d.T);
    const bool pair = item < np;
    // first channels of the item's two chunks; a copied item may have only its first chunk inside the head
    const int c0 = !pair ? d.rot + (item - np) * 2 * V : INTER ? item * 2 * V : item * V;
    const int c1 = pair && !INTER ? c0 + (d.rot >> 1) : c0 + V;
    const bool two = pair || c1 < d.D;
    float sn[V], cs[V];
    if (pair) {
        const int64_t po = (int64_t)b * d.pos_sB + (int64_t)t * d.pos_sT;
        const double pos = d.pos64 ? (double)G<const int64_t>(d.pos)[po] : (double)G<const int32_t>(d.pos)[po];
        const MEP_G double* fr = G<const double>(d.freqs) + item * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double turns = pos * (fr[j] * 0.15915494309189535);   // 1 / (2 pi)
            const double q = __builtin_rint(turns * 4.0);
            float s, c;
            sincos_turns((float)fma(q, -0.25, turns), s, c);
            const double k = fma(__builtin_floor(q * 0.25), -4.0, q);    // the quarter turn, 0 .. 3
            const bool odd = k == 1.0 || k == 3.0;
            const float s1 = odd ? c : s, c1v = odd ? s : c;
            sn[j] = (k >= 2.0 ? -s1 : s1) * (d.inverse ? -d.amplitude : d.amplitude);
            cs[j] = (k == 1.0 || k == 2.0 ? -c1v : c1v) * d.amplitude;
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (!d.x[w]) break;
        const MEP_G T* xb = G<const T>(d.x[w]) + (int64_t)b * d.sB[w] + (int64_t)t * d.sT[w];
        MEP_G T* yb = G<T>(d.y[w]) + tok * d.H[w] * d.M[w] * (int64_t)d.D;
        const int n = d.H[w] * d.M[w];
        // the heads of this thread: every hsplit-th, from hs
#pragma unroll 4
        for (int i = hs; i < n; i += hsplit) {
            const int h = d.M[w] == 1 ? i : i / d.M[w], m = d.M[w] == 1 ? 0 : i - h * d.M[w];
            const MEP_G T* xr = xb + (int64_t)h * d.sH[w] + (int64_t)m * d.sM[w];
            MEP_G T* yr = yb + (int64_t)i * d.D;
            float a[V], e[V];
            load_f32<T, V>(xr + c0, a);
            if (two) load_f32<T, V>(xr + c1, e);
            if (pair) {
                float u[V], v[V];
                if constexpr (INTER && V > 1) {   // pair j: elements 2j, 2j + 1 of the two chunks taken as one
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float p = 2 * j < V ? a[(2 * j) % V] : e[(2 * j) % V];
                        const float q = 2 * j + 1 < V ? a[(2 * j + 1) % V] : e[(2 * j + 1) % V];
                        const float r0 = p * cs[j] - q * sn[j], r1 = q * cs[j] + p * sn[j];
                        if (2 * j < V) { u[(2 * j) % V] = r0; u[(2 * j + 1) % V] = r1; }
                        else { v[(2 * j) % V] = r0; v[(2 * j + 1) % V] = r1; }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        u[j] = a[j] * cs[j] - e[j] * sn[j];
                        v[j] = e[j] * cs[j] + a[j] * sn[j];
                    }
                }
                store_f32<T, V>(yr + c0, u);
                store_f32<T, V>(yr + c1, v);
            } else {
                store_f32<T, V>(yr + c0, a);
                if (two) store_f32<T, V>(yr + c1, e);
            }
        }
    }
}

// false: more threads than a grid holds
template <int TYPE, int V>
bool launch_rotary(const mep_rotary_desc& d, hipStream_t st) {
    const int np = d.rot / 2 / V;                                    // V divides rot / 2 (fits)
    const int ni = np + (d.D - d.rot + 2 * V - 1) / (2 * V);
    const int64_t tok = (int64_t)d.B * d.T;
    const int heads = d.H[0] * d.M[0] > d.H[1] * d.M[1] || !d.x[1] ? d.H[0] * d.M[0] : d.H[1] * d.M[1];
    // split the heads until two rounds of 32 waves per compute unit are there (1,048,576 threads), at most one head each: with more
    // the sines are formed too often, with less the loads of a walk are too few in flight (32768 tokens of 20 heads: 88 us with 262,144
    // or 524,288 threads, 73, 81 with 2,621,440)
    int64_t hsplit = 1048576 / (tok * ni);
    hsplit = hsplit < 1 ? 1 : hsplit > heads ? heads : hsplit;
    if (tok * ni * hsplit >= (int64_t)1 << 32) return false;
    const int64_t blocks = (tok * ni * hsplit + ROT_THREADS - 1) / ROT_THREADS;
    if (d.interleaved) hipLaunchKernelGGL((k_rotary<TYPE, V, true>), dim3((unsigned)blocks), dim3(ROT_THREADS), 0, st, d, np, ni, (int)hsplit);
    else hipLaunchKernelGGL((k_rotary<TYPE, V, false>), dim3((unsigned)blocks), dim3(ROT_THREADS), 0, st, d, np, ni, (int)hsplit);
    return true;
}

// every chunk of V elements of the item layout lies inside its part of the head (its address need not be aligned)
bool fits(const mep_rotary_desc& d, int V) { return (d.rot / 2) % V == 0 && d.D % V == 0; }

template <int TYPE>
bool dispatch_rotary(const mep_rotary_desc& d, hipStream_t st) {
    if (TYPE != MEP_F32 && fits(d, 8)) return launch_rotary<TYPE, TYPE == MEP_F32 ? 4 : 8>(d, st);
    if (fits(d, 4)) return launch_rotary<TYPE, 4>(d, st);
    if (fits(d, 2)) return launch_rotary<TYPE, 2>(d, st);
    return launch_rotary<TYPE, 1>(d, st);
}

}  // namespace

extern "C" int mep_rotary(const mep_rotary_desc* desc, mep_stream_t stream) {
    if (!desc) { mep_set_error("mep_rotary: no descriptor"); return MEP_EINVAL; }
    const mep_rotary_desc& d = *desc;
    const int64_t tok = (int64_t)d.B * d.T;
    bool ok = d.B >= 0 && d.T >= 0 && d.D > 0 && d.rot >= 2 && d.rot % 2 == 0 && d.rot <= d.D && d.x[0] && d.y[0] &&
              d.freqs && d.pos && d.type >= MEP_F32 && d.type <= MEP_F16;
    for (int w = 0; w < 2 && ok; ++w)
        ok = !d.x[w] || (d.y[w] && d.H[w] > 0 && d.M[w] > 0 && (int64_t)d.H[w] * d.M[w] < (1 << 20));
    ok = ok && tok < ((int64_t)1 << 40);
    if (!ok) { mep_set_error("mep_rotary: invalid descriptor"); return MEP_EINVAL; }
    if (tok == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    ok = d.type == MEP_F32 ? dispatch_rotary<MEP_F32>(d, st)
         : d.type == MEP_BF16 ? dispatch_rotary<MEP_BF16>(d, st) : dispatch_rotary<MEP_F16>(d, st);
    if (!ok) { mep_set_error("mep_rotary: too many elements for one launch"); return MEP_EINVAL; }
    return mep_check_launch("mep_rotary");
}
