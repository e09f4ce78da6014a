// Group normalisation with an activation over channels-last tensors, forward and backward.
//
//   x (B, N, C): N pixels, C channels in G groups of cpg = C / G neighbours.  Per sample and group
//     mean = avg x,  rstd = 1 / sqrt(avg (x - mean)^2 + eps),  n = (x - mean) rstd,  z = n gamma_c + beta_c,  y = act(z)
//   backward, dz = dy act'(z):  dbeta_c = sum dz,  dgamma_c = sum dz n,
//     dx = rstd (dz gamma_c - S1 / cnt - n S2 / cnt),  S1 = sum over the group of dz gamma_c,  S2 of dz gamma_c n.
//
// All of it is bound by memory: the least it can move is one read and one write of the map (forward), two reads and one write
// (backward).  Two forms, chosen by size alone (gn_plan):
//   resident  a workgroup owns whole groups of one sample and keeps their values in registers (up to 8 vectors a thread
//             forward, 4 + 4 backward): every value is read once, mean and variance are two exact passes over registers.
//   slabs     the sample is cut into runs of pixels: one launch reduces them to partial statistics, the next joins the
//             partials of its sample (a few KB) and writes the result; the second read comes out of the last-level cache while
//             the map fits there.
// Measured (us on one MI355X; a 67 MB copy, which the last-level cache holds, runs at 7.2 TB/s, a 2 GB one at 5.05): resident, 32 x 32x32 x
// 256 bf16 in 32 groups: 14 forward (34 MB at 2.4 TB/s: one workgroup of 1024 threads a compute unit reads, reduces and writes in turn,
// nothing runs under the barriers), 15 + 4 backward; slabs, 32 x 128x128 x 64 in 16 groups with SiLU: 20 + 26 forward, 32 + 36 backward, 4.8 TB/s over
// the 537 MB that the four launches move (335 if each pass read its maps once, which needs a sample's workgroups to wait for each other).
// 16 and 8 vectors a thread instead of 8 and 4 spill; four workgroups a compute unit for the slabs' sums.
// Statistics never come from sums of squares: a thread's eight pixels give a mean and a sum of squared deviations, and these
// pairs are merged (Chan, Golub, LeVeque 1979), so a mean far from zero costs no digits.  Everything is summed in fp32 in an
// order that depends on the shape (and on whether the maps are 16-byte aligned) alone: results are the same from run to run.
#include "common.h"

namespace {

enum { ACT_NONE = 0, ACT_LRELU = 1, ACT_SILU = 2 };

template <typename T, int V> struct Vec;
template <> struct Vec<unsigned short, 8> {
    u32x4 r;
    __device__ __forceinline__ void load(const unsigned short* p) { r = *reinterpret_cast<const u32x4*>(p); }
    __device__ __forceinline__ void zero() { r = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ float get(int i) const { return (i & 1) ? bf16_hi(r[i >> 1]) : bf16_lo(r[i >> 1]); }
    static __device__ __forceinline__ void store(unsigned short* p, const float* f) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<u32x4*>(p) = o;
    }
};
template <> struct Vec<unsigned short, 1> {
    unsigned short r;
    __device__ __forceinline__ void load(const unsigned short* p) { r = *p; }
    __device__ __forceinline__ void zero() { r = 0; }
    __device__ __forceinline__ float get(int) const { return bf16_bits_to_f32(r); }
    static __device__ __forceinline__ void store(unsigned short* p, const float* f) { *p = f32_to_bf16_bits(f[0]); }
};
template <> struct Vec<float, 4> {
    f32x4 r;
    __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const f32x4*>(p); }
    __device__ __forceinline__ void zero() { r = f32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ float get(int i) const { return r[i]; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]}; }
};
template <> struct Vec<float, 1> {
    float r;
    __device__ __forceinline__ void load(const float* p) { r = *p; }
    __device__ __forceinline__ void zero() { r = 0.f; }
    __device__ __forceinline__ float get(int) const { return r; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *p = f[0]; }
};

struct GnArgs {
    const void* x; const void* dy; const float* gamma; const float* beta; void* out;
    float* mean; float* rstd;            // (B, G)
    float* part;                         // workspace
    float* dgamma; float* dbeta;
    int B, N, C, G, cpg;
    int cw, nc, pl;                      // channels a workgroup holds, vectors of a pixel's run of them, pixels side by side
    int slabs, slab_pixels, apply_wgs;
    float eps, slope;
};

// Groups of V neighbouring channels from c on: one division, then counted.
template <int V> __device__ __forceinline__ void groups_of(int (&g)[V], int c, int cpg) {
    int q = c / cpg, r = c - q * cpg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        g[i] = q;
        if (++r == cpg) { r = 0; ++q; }
    }
}
__device__ __forceinline__ float fast_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
template <int ACT> __device__ __forceinline__ float act_fwd(float z, float slope) {
    if (ACT == ACT_LRELU) return z > 0.f ? z : slope * z;
    if (ACT == ACT_SILU) return z * fast_sigmoid(z);
    return z;
}
template <int ACT> __device__ __forceinline__ float act_grad(float z, float slope) {
    if (ACT == ACT_LRELU) return z > 0.f ? 1.f : slope;
    if (ACT == ACT_SILU) { const float s = fast_sigmoid(z); return s * (1.f + z * (1.f - s)); }
    return 1.f;
}

// Sums of v[0..V) over the workgroup's pixel lanes: the channel sums end in red[0 .. cw).  Where the vectors of a pixel divide a wave, a
// wave adds up its own pixels with shuffles and a thread a channel adds the waves (two barriers; red: a row a wave); else by halves
// (red: a row a pixel lane).
template <int V> __device__ __forceinline__ void sum_over_pixels(float* red, const float* v, int p, int j, int pl, int cw, bool live) {
    const int nc = cw / V;
    if ((nc & (nc - 1)) == 0 && nc <= 64) {
        float w[V];
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = live ? v[i] : 0.f;
        for (int off = 32; off >= nc; off >>= 1)
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] += __shfl_xor(w[i], off, 64);
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
        if (lane < nc)
#pragma unroll
            for (int i = 0; i < V; ++i) red[wave * cw + lane * V + i] = w[i];
        __syncthreads();
        float s = 0.f;
        const int c = threadIdx.x;
        if (c < cw)
            for (int k = 0; k < waves; ++k) s += red[k * cw + c];
        float t[7];                                        // (cw <= 64 V = 512: one channel a thread of 64 .. 1024, more where threads are fewer)
        for (int e = 1; c + e * (int)blockDim.x < cw; ++e) {
            float q = 0.f;
            for (int k = 0; k < waves; ++k) q += red[k * cw + c + e * blockDim.x];
            t[e - 1] = q;
        }
        __syncthreads();
        if (c < cw) red[c] = s;
        for (int e = 1; c + e * (int)blockDim.x < cw; ++e) red[c + e * blockDim.x] = t[e - 1];
        __syncthreads();
        return;
    }
    if (live)
#pragma unroll
        for (int i = 0; i < V; ++i) red[p * cw + j * V + i] = v[i];
    __syncthreads();
    for (int n = pl; n > 1;) {
        const int half = (n + 1) >> 1;
        if (live && p < n - half)
#pragma unroll
            for (int i = 0; i < V; ++i) red[p * cw + j * V + i] += red[(p + half) * cw + j * V + i];
        n = half;
        __syncthreads();
    }
}

// Sum of ch[g * cpg .. + cpg) (LDS) for every group of the workgroup -> out[g] (LDS): a thread a group while that is a few adds, else a
// wave a group in turn.
__device__ __forceinline__ void sum_over_group(const float* ch, float* out, int groups, int cpg) {
    const int lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    if (cpg <= 32) {
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            float s = 0.f;
            for (int i = 0; i < cpg; ++i) s += ch[g * cpg + i];
            out[g] = s;
        }
    } else {
        for (int g = threadIdx.x >> 6; g < groups; g += nw) {
            float s = 0.f;
            for (int i = lane; i < cpg; i += 64) s += ch[g * cpg + i];
            s = wave_sum(s);
            if (lane == 0) out[g] = s;
        }
    }
    __syncthreads();
}

// ---- resident form ------------------------------------------------------------------------------------------------------
// Workgroups go round the 8 XCDs: each XCD gets the channel runs of the same samples, whose lines (two runs each) its L2 then reads once
// (32 x 32x32 x 256: forward 16.4 -> 15.2 us, backward 20.4 -> 15.7).
__device__ __forceinline__ int sample_run() {
    const int id = blockIdx.y * gridDim.x + blockIdx.x, total = gridDim.x * gridDim.y, q = total >> 3, r = total & 7, x = id & 7;
    return x * q + min(x, r) + (id >> 3);
}

template <typename T, int V, int E, int ACT>
__global__ __launch_bounds__(1024) void gn_fwd_resident(GnArgs a) {
    extern __shared__ float lds[];                        // red (pl * cw) | per group: mean, rstd
    float* red = lds;
    float* gm = lds + a.pl * a.cw;
    float* gr = gm + a.cw / a.cpg;
    const int groups = a.cw / a.cpg;
    const int id = sample_run(), b = id / gridDim.x, c0 = id % gridDim.x * a.cw;
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    const bool live = p < a.pl;
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.N * a.C + c0 + j * V;
    Vec<T, V> xs[E];
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = p + e * a.pl;
        if (live && n < a.N) xs[e].load(x + (int64_t)n * a.C);
        else xs[e].zero();
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += xs[e].get(i);
    sum_over_pixels<V>(red, acc, p, j, a.pl, a.cw, live);
    sum_over_group(red, gm, groups, a.cpg);
    const float inv = 1.f / ((float)a.N * (float)a.cpg);
    float mean[V], gamma[V], beta[V];
    int gi[V];
    groups_of<V>(gi, live ? j * V : 0, a.cpg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mean[i] = live ? gm[gi[i]] * inv : 0.f;
        gamma[i] = live ? a.gamma[c0 + j * V + i] : 0.f;
        beta[i] = live ? a.beta[c0 + j * V + i] : 0.f;
        acc[i] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (p + e * a.pl < a.N)
#pragma unroll
            for (int i = 0; i < V; ++i) { const float d = xs[e].get(i) - mean[i]; acc[i] += d * d; }
    sum_over_pixels<V>(red, acc, p, j, a.pl, a.cw, live);
    sum_over_group(red, gr, groups, a.cpg);
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        const int64_t o = (int64_t)b * a.G + c0 / a.cpg + g;
        const float r = 1.f / sqrtf(gr[g] * inv + a.eps);
        a.mean[o] = gm[g] * inv;
        a.rstd[o] = r;
        gr[g] = r;
    }
    __syncthreads();
    if (!live) return;
    float scale[V];
#pragma unroll
    for (int i = 0; i < V; ++i) scale[i] = gr[gi[i]];
    T* y = reinterpret_cast<T*>(a.out) + (int64_t)b * a.N * a.C + c0 + j * V;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = p + e * a.pl;
        if (n >= a.N) break;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = act_fwd<ACT>((xs[e].get(i) - mean[i]) * scale[i] * gamma[i] + beta[i], a.slope);
        Vec<T, V>::store(y + (int64_t)n * a.C, f);
    }
}

// part: (B, C, 2) channel sums (dz, dz n), reduced over B by gn_param_grads.
template <typename T, int V, int E, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_resident(GnArgs a) {
    extern __shared__ float lds[];                        // red (pl * cw) | s1 (groups) | s2 (groups)
    float* red = lds;
    const int groups = a.cw / a.cpg;
    float* s1 = lds + a.pl * a.cw;
    float* s2 = s1 + groups;
    const int id = sample_run(), b = id / gridDim.x, c0 = id % gridDim.x * a.cw;
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    const bool live = p < a.pl;
    const int64_t base = (int64_t)b * a.N * a.C + c0 + j * V;
    const T* x = reinterpret_cast<const T*>(a.x) + base;
    const T* dy = reinterpret_cast<const T*>(a.dy) + base;
    Vec<T, V> xs[E], ds[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = p + e * a.pl;
        if (live && n < a.N) { xs[e].load(x + (int64_t)n * a.C); ds[e].load(dy + (int64_t)n * a.C); }
        else { xs[e].zero(); ds[e].zero(); }
    }
    float mean[V], rstd[V], gamma[V], beta[V], sa[V], sb[V];
    int gi[V];
    groups_of<V>(gi, live ? j * V : 0, a.cpg);
    const int64_t g0 = (int64_t)b * a.G + c0 / a.cpg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = c0 + (live ? j * V + i : 0);
        mean[i] = a.mean[g0 + gi[i]];
        rstd[i] = a.rstd[g0 + gi[i]];
        gamma[i] = a.gamma[c];
        beta[i] = a.beta[c];
        sa[i] = sb[i] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (p + e * a.pl < a.N)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n = (xs[e].get(i) - mean[i]) * rstd[i];
                const float dz = ds[e].get(i) * act_grad<ACT>(n * gamma[i] + beta[i], a.slope);
                sa[i] += dz;
                sb[i] += dz * n;
            }
    sum_over_pixels<V>(red, sa, p, j, a.pl, a.cw, live);
    for (int c = threadIdx.x; c < a.cw; c += blockDim.x) {
        a.part[2 * ((int64_t)b * a.C + c0 + c)] = red[c];
        red[c] *= a.gamma[c0 + c];
    }
    __syncthreads();
    sum_over_group(red, s1, groups, a.cpg);
    sum_over_pixels<V>(red, sb, p, j, a.pl, a.cw, live);
    for (int c = threadIdx.x; c < a.cw; c += blockDim.x) {
        a.part[2 * ((int64_t)b * a.C + c0 + c) + 1] = red[c];
        red[c] *= a.gamma[c0 + c];
    }
    __syncthreads();
    sum_over_group(red, s2, groups, a.cpg);
    if (!live) return;
    const float inv = 1.f / ((float)a.N * (float)a.cpg);
    float m1[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { m1[i] = s1[gi[i]] * inv; m2[i] = s2[gi[i]] * inv; }
    T* dx = reinterpret_cast<T*>(a.out) + base;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = p + e * a.pl;
        if (n >= a.N) break;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float nh = (xs[e].get(i) - mean[i]) * rstd[i];
            const float dz = ds[e].get(i) * act_grad<ACT>(nh * gamma[i] + beta[i], a.slope);
            f[i] = rstd[i] * (dz * gamma[i] - m1[i] - nh * m2[i]);
        }
        Vec<T, V>::store(dx + (int64_t)n * a.C, f);
    }
}

// ---- slab form ----------------------------------------------------------------------------------------------------------
// part: (B, slabs, G, 2): mean and sum of squared deviations of a slab's share of a group.
template <typename T, int V>
__global__ __launch_bounds__(1024) void gn_slab_stats(GnArgs a) {
    extern __shared__ float lds[];                        // mean (pl * C) | m2 (pl * C)
    float* lm = lds;
    float* lq = lds + a.pl * a.C;
    const int b = blockIdx.y, s = blockIdx.x;
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    const bool live = p < a.pl;
    const int n0 = s * a.slab_pixels, n1 = min(a.N, n0 + a.slab_pixels);
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.N * a.C + j * V;
    float mean[V], m2[V];
    float cnt = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    constexpr int U = 8;
    if (live)
        for (int n = n0 + p; n < n1; n += U * a.pl) {
            Vec<T, V> xs[U];
            int k = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (n + u * a.pl < n1) { xs[u].load(x + (int64_t)(n + u * a.pl) * a.C); ++k; }
                else xs[u].zero();
            const float kf = (float)k, ik = 1.f / kf, tot = cnt + kf;
            const float wb = kf / tot, wq = cnt * wb;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float sum = 0.f, q = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) sum += xs[u].get(i);
                const float mb = sum * ik;
#pragma unroll
                for (int u = 0; u < U; ++u) { const float d = u < k ? xs[u].get(i) - mb : 0.f; q += d * d; }
                const float d = mb - mean[i];
                mean[i] += d * wb;
                m2[i] += q + d * d * wq;
            }
            cnt = tot;
        }
    if (live)
#pragma unroll
        for (int i = 0; i < V; ++i) { lm[p * a.C + j * V + i] = mean[i]; lq[p * a.C + j * V + i] = m2[i]; }
    __syncthreads();
    // a wave per group in turn: the (pixel lane, channel) pairs of the group, each with the count of its pixel lane
    const int lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    const int rows = n1 - n0;
    const float total = (float)rows * (float)a.cpg;
    for (int g = threadIdx.x >> 6; g < a.G; g += nw) {
        float sum = 0.f;
        for (int e = lane; e < a.pl * a.cpg; e += 64) {
            const int pp = e / a.cpg, c = e - pp * a.cpg;
            const float k = (float)((rows - pp + a.pl - 1) / a.pl);          // pixels of lane pp in this slab (>= 0: rows >= 1, pp < pl)
            sum += k * lm[pp * a.C + g * a.cpg + c];
        }
        const float m = wave_sum(sum) / total;
        float q = 0.f;
        for (int e = lane; e < a.pl * a.cpg; e += 64) {
            const int pp = e / a.cpg, c = e - pp * a.cpg;
            const float k = (float)((rows - pp + a.pl - 1) / a.pl);
            const float d = lm[pp * a.C + g * a.cpg + c] - m;
            q += lq[pp * a.C + g * a.cpg + c] + k * d * d;
        }
        q = wave_sum(q);
        if (lane == 0) {
            float* o = a.part + 2 * (((int64_t)b * a.slabs + s) * a.G + g);
            o[0] = m;
            o[1] = q;
        }
    }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(1024) void gn_slab_apply(GnArgs a) {
    extern __shared__ float lds[];                        // mean (G) | rstd (G)
    float* gm = lds;
    float* gr = lds + a.G;
    const int b = blockIdx.y;
    const int lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    const float inv = 1.f / ((float)a.N * (float)a.cpg);
    for (int g = threadIdx.x >> 6; g < a.G; g += nw) {
        const float* pt = a.part + 2 * ((int64_t)b * a.slabs * a.G + g);
        float sum = 0.f;
        for (int s = lane; s < a.slabs; s += 64)
            sum += (float)min(a.slab_pixels, a.N - s * a.slab_pixels) * pt[(int64_t)2 * s * a.G];
        const float m = wave_sum(sum) / (float)a.N;
        float q = 0.f;
        for (int s = lane; s < a.slabs; s += 64) {
            const float k = (float)min(a.slab_pixels, a.N - s * a.slab_pixels) * (float)a.cpg;
            const float d = pt[(int64_t)2 * s * a.G] - m;
            q += pt[(int64_t)2 * s * a.G + 1] + k * d * d;
        }
        q = wave_sum(q);
        if (lane == 0) {
            const float r = 1.f / sqrtf(q * inv + a.eps);
            gm[g] = m;
            gr[g] = r;
            if (blockIdx.x == 0) { a.mean[(int64_t)b * a.G + g] = m; a.rstd[(int64_t)b * a.G + g] = r; }
        }
    }
    __syncthreads();
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    if (p >= a.pl) return;
    float sc[V], sh[V];
    int gi[V];
    groups_of<V>(gi, j * V, a.cpg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = j * V + i, g = gi[i];
        sc[i] = gr[g] * a.gamma[c];
        sh[i] = gm[g];
    }
    float beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) beta[i] = a.beta[j * V + i];
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.N * a.C + j * V;
    T* y = reinterpret_cast<T*>(a.out) + (int64_t)b * a.N * a.C + j * V;
    constexpr int U = 4;
    const int step = a.pl * gridDim.x;
    for (int n = blockIdx.x * a.pl + p; n < a.N; n += U * step) {
        Vec<T, V> xs[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (n + u * step < a.N) xs[u].load(x + (int64_t)(n + u * step) * a.C);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (n + u * step < a.N) {
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = act_fwd<ACT>((xs[u].get(i) - sh[i]) * sc[i] + beta[i], a.slope);
                Vec<T, V>::store(y + (int64_t)(n + u * step) * a.C, f);
            }
    }
}

// part: (B, slabs, C, 2) channel sums (dz, dz n), then (B, slabs, G, 2) group sums of them times gamma.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(1024) void gn_slab_bwd_sums(GnArgs a) {
    extern __shared__ float lds[];                        // red (pl * C)
    float* red = lds;
    const int b = blockIdx.y, s = blockIdx.x;
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    const bool live = p < a.pl;
    const int n0 = s * a.slab_pixels, n1 = min(a.N, n0 + a.slab_pixels);
    const int64_t base = (int64_t)b * a.N * a.C + j * V;
    const T* x = reinterpret_cast<const T*>(a.x) + base;
    const T* dy = reinterpret_cast<const T*>(a.dy) + base;
    float mean[V], rstd[V], gamma[V], beta[V], sa[V], sb[V];
    int gi[V];
    groups_of<V>(gi, live ? j * V : 0, a.cpg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = live ? j * V + i : 0;
        mean[i] = a.mean[(int64_t)b * a.G + gi[i]];
        rstd[i] = a.rstd[(int64_t)b * a.G + gi[i]];
        gamma[i] = a.gamma[c];
        beta[i] = a.beta[c];
        sa[i] = sb[i] = 0.f;
    }
    constexpr int U = 4;
    if (live)
        for (int n = n0 + p; n < n1; n += U * a.pl) {
            Vec<T, V> xs[U], ds[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (n + u * a.pl < n1) {
                    xs[u].load(x + (int64_t)(n + u * a.pl) * a.C);
                    ds[u].load(dy + (int64_t)(n + u * a.pl) * a.C);
                } else { xs[u].zero(); ds[u].zero(); }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (n + u * a.pl < n1)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float nh = (xs[u].get(i) - mean[i]) * rstd[i];
                        const float dz = ds[u].get(i) * act_grad<ACT>(nh * gamma[i] + beta[i], a.slope);
                        sa[i] += dz;
                        sb[i] += dz * nh;
                    }
        }
    const int64_t row = (int64_t)b * a.slabs + s;
    float* cp = a.part + 2 * row * a.C;
    float* gp = a.part + 2 * (int64_t)a.B * a.slabs * a.C + 2 * row * a.G;
    const int lane = threadIdx.x & 63, nw = blockDim.x >> 6;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        sum_over_pixels<V>(red, w ? sb : sa, p, j, a.pl, a.C, live);
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) cp[2 * c + w] = red[c];
        for (int g = threadIdx.x >> 6; g < a.G; g += nw) {
            float t = 0.f;
            for (int i = lane; i < a.cpg; i += 64) t += red[g * a.cpg + i] * a.gamma[g * a.cpg + i];
            t = wave_sum(t);
            if (lane == 0) gp[2 * g + w] = t;
        }
        __syncthreads();
    }
}

// dgamma / dbeta of 8 channels from `rows` partial rows of (C, 2): a row lane for every 16 threads, eight rows at a time, joined in a fixed
// order.
constexpr int PG = 8;
__device__ void param_grads(const float* part, int64_t rows, int C, int c0, float* dgamma, float* dbeta, float* red) {
    const int col = threadIdx.x & 15;                      // (channel, which) of 8 channels
    const int lanes = blockDim.x >> 4, r0 = threadIdx.x >> 4;
    const bool in = c0 * 2 + col < 2 * C;
    float s = 0.f;
    if (in)
        for (int64_t r = r0; r < rows; r += 8 * lanes) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t q = r + k * lanes;
                v[k] = part[(q < rows ? q : rows - 1) * 2 * C + c0 * 2 + col];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s += r + k * lanes < rows ? v[k] : 0.f;
        }
    red[threadIdx.x] = s;
    __syncthreads();
    if (r0 == 0 && in) {
        for (int k = 1; k < lanes; ++k) s += red[k * 16 + col];
        if (col & 1) dgamma[c0 + (col >> 1)] = s;
        else dbeta[c0 + (col >> 1)] = s;
    }
}

__global__ __launch_bounds__(256) void gn_param_grads(const float* part, int64_t rows, int C, float* dgamma, float* dbeta) {
    __shared__ float red[256];
    param_grads(part, rows, C, blockIdx.x * PG, dgamma, dbeta, red);
}

// grid.x = ceil(C / 8) workgroups that sum the parameters' gradients (of sample 0: a long chain of adds, so they start first), then
// apply_wgs that write dx.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(1024) void gn_slab_bwd_apply(GnArgs a) {
    extern __shared__ float lds[];                        // s1 (G) | s2 (G), or red (blockDim)
    const int b = blockIdx.y;
    const int first = (a.C + PG - 1) / PG;
    if ((int)blockIdx.x < first) {
        if (b == 0) param_grads(a.part, (int64_t)a.B * a.slabs, a.C, blockIdx.x * PG, a.dgamma, a.dbeta, lds);
        return;
    }
    const int wg = blockIdx.x - first;
    float* s1 = lds;
    float* s2 = lds + a.G;
    const int lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    const float* gp = a.part + 2 * (int64_t)a.B * a.slabs * a.C + 2 * (int64_t)b * a.slabs * a.G;
    const float inv = 1.f / ((float)a.N * (float)a.cpg);
    for (int g = threadIdx.x >> 6; g < a.G; g += nw) {
        float t1 = 0.f, t2 = 0.f;
        for (int s = lane; s < a.slabs; s += 64) {
            t1 += gp[2 * ((int64_t)s * a.G + g)];
            t2 += gp[2 * ((int64_t)s * a.G + g) + 1];
        }
        t1 = wave_sum(t1);
        t2 = wave_sum(t2);
        if (lane == 0) { s1[g] = t1 * inv; s2[g] = t2 * inv; }
    }
    __syncthreads();
    const int p = threadIdx.x / a.nc, j = threadIdx.x - p * a.nc;
    if (p >= a.pl) return;
    float mean[V], rstd[V], gamma[V], beta[V], m1[V], m2[V];
    int gi[V];
    groups_of<V>(gi, j * V, a.cpg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = j * V + i, g = gi[i];
        mean[i] = a.mean[(int64_t)b * a.G + g];
        rstd[i] = a.rstd[(int64_t)b * a.G + g];
        gamma[i] = a.gamma[c];
        beta[i] = a.beta[c];
        m1[i] = s1[g];
        m2[i] = s2[g];
    }
    const int64_t base = (int64_t)b * a.N * a.C + j * V;
    const T* x = reinterpret_cast<const T*>(a.x) + base;
    const T* dy = reinterpret_cast<const T*>(a.dy) + base;
    T* dx = reinterpret_cast<T*>(a.out) + base;
    constexpr int U = 4;
    const int step = a.pl * a.apply_wgs;
    for (int n = wg * a.pl + p; n < a.N; n += U * step) {
        Vec<T, V> xs[U], ds[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (n + u * step < a.N) {
                xs[u].load(x + (int64_t)(n + u * step) * a.C);
                ds[u].load(dy + (int64_t)(n + u * step) * a.C);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (n + u * step < a.N) {
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float nh = (xs[u].get(i) - mean[i]) * rstd[i];
                    const float dz = ds[u].get(i) * act_grad<ACT>(nh * gamma[i] + beta[i], a.slope);
                    f[i] = rstd[i] * (dz * gamma[i] - m1[i] - nh * m2[i]);
                }
                Vec<T, V>::store(dx + (int64_t)(n + u * step) * a.C, f);
            }
    }
}

// ---- which form, and its launch -----------------------------------------------------------------------------------------
int gcd_i(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

struct GnPlan { bool resident; int vec, cw, nc, pl, threads, e, slabs, slab_pixels, apply_wgs; };

// Resident where a workgroup can hold whole groups of a sample: at most `most` vectors a thread at 1024 threads.  The run of
// channels is the shortest of whole groups and whole vectors that reaches 64 bytes (half a cache line: narrower runs re-read
// lines, wider ones leave compute units idle).
GnPlan gn_plan(int B, int N, int C, int G, int esize, bool aligned, int most) {
    GnPlan p{};
    const int full = 16 / esize, cpg = C / G;
    p.vec = (C % full == 0 && aligned) ? full : 1;
    int unit = cpg / gcd_i(cpg, p.vec) * p.vec;             // lcm(cpg, vec): divides C, as both do
    p.cw = unit;
    while (p.cw * esize < 64 && p.cw < C) {
        int next = p.cw + unit;
        while (next < C && C % next) next += unit;
        p.cw = next;
    }
    p.nc = p.cw / p.vec;
    const int64_t vectors = (int64_t)N * p.nc;
    if (p.nc <= 1024 && vectors <= (int64_t)1024 * most && (int64_t)N <= (int64_t)(1024 / p.nc) * most) {
        p.resident = true;
        int t = 64;
        while (t < 1024 && (t < p.nc || (int64_t)t * 2 < vectors)) t *= 2;     // about two vectors a thread while there are threads
        p.threads = t;
        p.pl = t / p.nc;
        p.e = ceil_div(N, p.pl);
        if (p.e > most) { p.threads = 1024; p.pl = 1024 / p.nc; p.e = ceil_div(N, p.pl); }
        if (p.pl > N) p.pl = N;
        return p;
    }
    p.cw = C;
    p.nc = C / p.vec;
    p.threads = p.nc > 256 ? 1024 : 256;
    p.pl = p.threads / p.nc;
    if (p.pl > 0 && B > 0) {
        // about four workgroups a compute unit, at least 8 pixels for each pixel lane, at most 256 slabs a sample to join
        const int64_t want = (1024 + B - 1) / B;
        int64_t s = (N + (int64_t)p.pl * 8 - 1) / ((int64_t)p.pl * 8);
        if (s > want) s = want;
        if (s > 256) s = 256;
        if (s < 1) s = 1;
        p.slab_pixels = ceil_div(N, s);
        p.slabs = ceil_div(N, p.slab_pixels);
        int64_t ap = (N + (int64_t)p.pl * 4 - 1) / ((int64_t)p.pl * 4), cap = (2048 + B - 1) / B;
        p.apply_wgs = (int)(ap < cap ? ap : cap);
    }
    return p;
}

const int FWD_MOST = 8, BWD_MOST = 4;      // (16 and 8 vectors spill at the 128 registers that 1024 threads leave)

int gn_check(const void* x, int B, int N, int C, int G, int dtype, int act, const char* who) {
    RGBD_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype must be 0 (bf16) or 1 (fp32), got %d", who, dtype);
    RGBD_REQUIRE(act >= 0 && act <= 2, "%s: act must be 0 (none), 1 (leaky ReLU) or 2 (SiLU), got %d", who, act);
    RGBD_REQUIRE(B >= 0 && B <= 65535 && N >= 0 && N < (1 << 30) && C > 0 && G > 0 && C % G == 0,
                 "%s: bad sizes B=%d N=%d C=%d groups=%d (groups must divide C)", who, B, N, C, G);
    const int full = dtype ? 4 : 8;
    RGBD_REQUIRE(C <= (C % full == 0 && ((uintptr_t)x & 15) == 0 ? 1024 * full : 1024),
                 "%s: C=%d: at most %d channels, 1024 where 16-byte vectors do not fit", who, C, 1024 * full);
    return 0;
}

template <typename T, int V, int ACT> void launch_fwd(const GnPlan& p, GnArgs& a, hipStream_t s) {
    if (p.resident) {
        const dim3 grid(a.C / p.cw, a.B);
        const size_t lds = (size_t)(p.pl * p.cw + 2 * (p.cw / a.cpg)) * 4;
        if (p.e <= 2) hipLaunchKernelGGL((gn_fwd_resident<T, V, 2, ACT>), grid, dim3(p.threads), lds, s, a);
        else if (p.e <= 4) hipLaunchKernelGGL((gn_fwd_resident<T, V, 4, ACT>), grid, dim3(p.threads), lds, s, a);
        else hipLaunchKernelGGL((gn_fwd_resident<T, V, 8, ACT>), grid, dim3(p.threads), lds, s, a);
        return;
    }
    hipLaunchKernelGGL((gn_slab_stats<T, V>), dim3(a.slabs, a.B), dim3(p.threads), (size_t)2 * p.pl * a.C * 4, s, a);
    hipLaunchKernelGGL((gn_slab_apply<T, V, ACT>), dim3(a.apply_wgs, a.B), dim3(p.threads), (size_t)2 * a.G * 4, s, a);
}

template <typename T, int V, int ACT> void launch_bwd(const GnPlan& p, GnArgs& a, hipStream_t s) {
    if (p.resident) {
        const dim3 grid(a.C / p.cw, a.B);
        const size_t lds = (size_t)(p.pl * p.cw + 2 * (p.cw / a.cpg)) * 4;
        if (p.e <= 2) hipLaunchKernelGGL((gn_bwd_resident<T, V, 2, ACT>), grid, dim3(p.threads), lds, s, a);
        else hipLaunchKernelGGL((gn_bwd_resident<T, V, 4, ACT>), grid, dim3(p.threads), lds, s, a);
        hipLaunchKernelGGL(gn_param_grads, dim3(ceil_div(a.C, PG)), dim3(256), 0, s, a.part, (int64_t)a.B, a.C, a.dgamma, a.dbeta);
        return;
    }
    hipLaunchKernelGGL((gn_slab_bwd_sums<T, V, ACT>), dim3(a.slabs, a.B), dim3(p.threads), (size_t)p.pl * a.C * 4, s, a);
    const size_t lds = (size_t)(2 * a.G > p.threads ? 2 * a.G : p.threads) * 4;
    hipLaunchKernelGGL((gn_slab_bwd_apply<T, V, ACT>), dim3(a.apply_wgs + ceil_div(a.C, PG), a.B), dim3(p.threads), lds, s, a);
}

template <typename T, int V> void by_act(bool bwd, int act, const GnPlan& p, GnArgs& a, hipStream_t s) {
    if (act == ACT_NONE) bwd ? launch_bwd<T, V, ACT_NONE>(p, a, s) : launch_fwd<T, V, ACT_NONE>(p, a, s);
    else if (act == ACT_LRELU) bwd ? launch_bwd<T, V, ACT_LRELU>(p, a, s) : launch_fwd<T, V, ACT_LRELU>(p, a, s);
    else bwd ? launch_bwd<T, V, ACT_SILU>(p, a, s) : launch_fwd<T, V, ACT_SILU>(p, a, s);
}

void gn_dispatch(bool bwd, int dtype, int act, const GnPlan& p, GnArgs& a, hipStream_t s) {
    a.cw = p.cw; a.nc = p.nc; a.pl = p.pl; a.slabs = p.slabs; a.slab_pixels = p.slab_pixels; a.apply_wgs = p.apply_wgs;
    if (dtype == 0) p.vec == 8 ? by_act<unsigned short, 8>(bwd, act, p, a, s) : by_act<unsigned short, 1>(bwd, act, p, a, s);
    else p.vec == 4 ? by_act<float, 4>(bwd, act, p, a, s) : by_act<float, 1>(bwd, act, p, a, s);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int64_t rgbd_group_norm_workspace(int B, int N, int C, int groups, int dtype, int backward) {
    if (gn_check(nullptr, B, N, C, groups, dtype, 0, "rgbd_group_norm_workspace")) return -1;
    // the vector and the scalar form cut a sample differently: room for either
    int64_t most = backward ? 1 : 0;
    for (int al = 0; al < 2; ++al) {
        const GnPlan p = gn_plan(B, N, C, groups, dtype ? 4 : 2, al != 0, backward ? BWD_MOST : FWD_MOST);
        const int64_t f = backward ? (p.resident ? (int64_t)2 * B * C : (int64_t)2 * B * p.slabs * (C + groups))
                                   : (p.resident ? 0 : (int64_t)2 * B * p.slabs * groups);
        if (f > most) most = f;
    }
    return most;
}

extern "C" int rgbd_group_norm_fwd(const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                                   float* workspace, int B, int N, int C, int groups, int dtype, int act, float eps, float slope,
                                   void* stream) {
    if (gn_check(x, B, N, C, groups, dtype, act, "rgbd_group_norm_fwd")) return -1;
    if (B == 0 || N == 0) return 0;
    RGBD_REQUIRE(x && gamma && beta && y && mean && rstd, "rgbd_group_norm_fwd: null pointer");
    RGBD_REQUIRE(eps >= 0.f, "rgbd_group_norm_fwd: eps must not be negative");
    const GnPlan p = gn_plan(B, N, C, groups, dtype ? 4 : 2, aligned16(x) && aligned16(y), FWD_MOST);
    RGBD_REQUIRE(p.pl > 0, "rgbd_group_norm_fwd: C=%d does not fit a workgroup", C);
    RGBD_REQUIRE(p.resident || workspace, "rgbd_group_norm_fwd: null workspace");
    GnArgs a{};
    a.x = x; a.gamma = gamma; a.beta = beta; a.out = y; a.mean = mean; a.rstd = rstd; a.part = workspace;
    a.B = B; a.N = N; a.C = C; a.G = groups; a.cpg = C / groups; a.eps = eps; a.slope = slope;
    gn_dispatch(false, dtype, act, p, a, (hipStream_t)stream);
    RGBD_CHECK_LAUNCH("rgbd_group_norm_fwd");
    return 0;
}

extern "C" int rgbd_group_norm_bwd(const void* x, const void* dy, const float* gamma, const float* beta, const float* mean,
                                   const float* rstd, void* dx, float* dgamma, float* dbeta, float* workspace, int B, int N, int C,
                                   int groups, int dtype, int act, float slope, void* stream) {
    if (gn_check(x, B, N, C, groups, dtype, act, "rgbd_group_norm_bwd")) return -1;
    RGBD_REQUIRE(gamma && dgamma && dbeta, "rgbd_group_norm_bwd: null pointer");
    if (B == 0 || N == 0) {
        hipError_t e = rgbd_zero_async(dgamma, (size_t)C * 4, (hipStream_t)stream);
        if (e == hipSuccess) e = rgbd_zero_async(dbeta, (size_t)C * 4, (hipStream_t)stream);
        RGBD_REQUIRE(e == hipSuccess, "rgbd_group_norm_bwd: %s", hipGetErrorString(e));
        return 0;
    }
    RGBD_REQUIRE(x && dy && beta && mean && rstd && dx && workspace, "rgbd_group_norm_bwd: null pointer");
    const GnPlan p = gn_plan(B, N, C, groups, dtype ? 4 : 2, aligned16(x) && aligned16(dy) && aligned16(dx), BWD_MOST);
    RGBD_REQUIRE(p.pl > 0, "rgbd_group_norm_bwd: C=%d does not fit a workgroup", C);
    GnArgs a{};
    a.x = x; a.dy = dy; a.gamma = gamma; a.beta = beta; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.out = dx; a.part = workspace; a.dgamma = dgamma; a.dbeta = dbeta;
    a.B = B; a.N = N; a.C = C; a.G = groups; a.cpg = C / groups; a.slope = slope;
    gn_dispatch(true, dtype, act, p, a, (hipStream_t)stream);
    RGBD_CHECK_LAUNCH("rgbd_group_norm_bwd");
    return 0;
}
