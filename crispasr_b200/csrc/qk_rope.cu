// qk_rope.cu — the pass between the projections of a decoder layer and its attention: norm of every query and key head,
// rotation by position, and K and V into the cache rows.
//
// For a row x of a head at position p:  y = x * w / sqrt(mean(x^2) + eps), then every pair (y_a, y_b) of the rotated values turns
// by t_i = p * scale * base^(-2i/n).  As graph nodes these are two norms, two products, two rotations and two writes into the
// cache, each of which reads and writes every row; here a row is read once and written once, so the pass is bound by its bytes
// where many rows enter and by the launch where one does.
#include <cmath>
#include <cstring>
#include <type_traits>

#include "kv_cache.h"
#include "kv_rows.cuh"

namespace b200 {
namespace {

constexpr int kMaxHalf = 64;   // pairs of a head of 128
constexpr int kRopeWarps = 4;

struct RopeArgs {
    const uint8_t* src[3];   // q, k, v; a tensor that is not there has no heads
    int64_t snb1[3], snb2[3], snb3[3];
    uint8_t* dst[3];         // q_out and k_out, or the cache rows of K and V
    int64_t dnb1[3], dnb2[3], dnb3[3];
    int heads[3];
    const float* w[2];       // norm weights of q and k; null = no norm
    int n, hd, n_dims, neox, out_f32, ctx_rows, pos0, chunks;   // chunks: warps per token
    int n_tokens;            // streams x rows
    float eps, inv_hd;
    const int32_t* pos;
    const int32_t* n_rows;
    uint64_t turns[kMaxHalf];   // turns per position of each pair, as a fraction of 2^64
};

// Angles: `turns` counts the turn of a pair per position in units of 2^-64 turns, and the product with the position wraps at
// whole turns, so the reduction of a far position's angle is exact (in fp32 the angle at position 100 000 is off by 4e-3).
// The 32 high bits as a signed number are the angle in (-pi, pi] to 2^-31 of pi; sincospif takes it from there.
__device__ __forceinline__ void angle_of(uint64_t turns, int64_t p, float& c, float& s) {
    sincospif((float)(int32_t)((turns * (uint64_t)p) >> 32) * 0x1p-31f, &s, &c);
}

template <bool F32, bool V16>
__device__ __forceinline__ void load_in8(const uint8_t* p, float (&f)[8]) {
    if constexpr (F32 && V16) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = load_global(reinterpret_cast<const float*>(p) + i);
    } else {
        uint32_t u[4];
        if constexpr (V16) {
            const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p));
            u[0] = x.x, u[1] = x.y, u[2] = x.z, u[3] = x.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                u[i] = load_global(reinterpret_cast<const uint16_t*>(p) + 2 * i) | (uint32_t)load_global(reinterpret_cast<const uint16_t*>(p) + 2 * i + 1) << 16;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            f[2 * i] = x.x, f[2 * i + 1] = x.y;
        }
    }
}

// Four values of either half of a row (16-byte aligned rows).
template <bool F32>
__device__ __forceinline__ void load_in4x2(const uint8_t* p, const uint8_t* q, float (&f)[8]) {
    if constexpr (F32) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(q));
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p)), b = __ldcs(reinterpret_cast<const uint2*>(q));
        const uint32_t u[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            f[2 * i] = x.x, f[2 * i + 1] = x.y;
        }
    }
}
__device__ __forceinline__ void store_out4x2(uint8_t* row, int c, const float (&f)[8], int hd, int f32) {
#pragma unroll
    for (int part = 0; part < 2; part++) {
        const float* x = f + 4 * part;
        const int e = c + part * (hd / 2);
        if (f32) *reinterpret_cast<float4*>(row + 4 * e) = make_float4(x[0], x[1], x[2], x[3]);
        else *reinterpret_cast<uint2*>(row + 2 * e) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    }
}
template <bool V16>
__device__ __forceinline__ void store_out8(uint8_t* p, const float (&f)[8], int f32) {
    if (f32) store8<true, V16>(p, f);
    else store8<false, V16>(p, f);
}

// A warp takes one token and a run of its rows (the heads of q, then those of k, then of v), eight values per lane, 32 / LPR rows at
// a time, the loads of U such groups in flight: the cosines and sines of the token's position are worked out once for all of them, the norm's
// weights once per tensor.
// LPR: lanes per row, hd / 8 rounded up to a power of two.  CACHE: type of the cache, or F32 for outputs that are tensors.
// HALVES (NEOX, all of a head of 64 or 128 rotated, 16-byte rows): a lane has four values of either half of its row, which are each
// other's partners: no exchange between lanes, half as many cosines, and 256 contiguous bytes per load of a row.  Otherwise a lane has eight
// consecutive values, and with NEOX fetches the partners from another lane.
template <bool F32, bool V16, int LPR, int CACHE, bool HALVES>
__global__ void __launch_bounds__(32 * kRopeWarps) qk_rope_kernel(const __grid_constant__ RopeArgs a) {
    let_dependents_launch();
    __shared__ uint64_t s_turns[kMaxHalf];
    if (threadIdx.x < a.n_dims / 2) s_turns[threadIdx.x] = a.turns[threadIdx.x];
    __syncthreads();
    constexpr int RPW = 32 / LPR, ES = F32 ? 4 : 2, U = is_blocks(CACHE) ? 2 : 4;   // groups in flight: block arithmetic wants the registers of two
    const int lane = threadIdx.x & 31, sub = lane / LPR, l = lane % LPR, half = a.n_dims / 2;
    const int c = HALVES ? 4 * l : 8 * l;   // the lane's first value
    const int64_t unit = (int64_t)blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
    const int token = (int)(unit / a.chunks), chunk = (int)(unit - (int64_t)token * a.chunks);
    // launched with programmatic stream serialisation: nothing is read before the kernels ahead of this one have completed
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (token >= a.n_tokens) return;   // (whole warps)
    const int s = token / a.n, i = token - s * a.n;
    const int64_t p = (int64_t)(a.pos ? a.pos[s] : a.pos0) + i;
    const bool valid = !a.n_rows || i < a.n_rows[s];
    const bool stored = p >= 0 && p < a.ctx_rows;

    int groups[3], total = 0;
#pragma unroll
    for (int x = 0; x < 3; x++) groups[x] = (a.heads[x] + RPW - 1) / RPW, total += groups[x];
    const int per = (total + a.chunks - 1) / a.chunks, lo = chunk * per, hi = min(total, lo + per);
    const bool inside = c < a.hd;   // (a head of 96 or 80 leaves some of the sixteen lanes without values)

    if (!valid) {   // a row behind n_rows: zeros to the tensors, nothing to the cache
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kind = 0; kind < (CACHE == B200_TYPE_F32 ? 2 : 1); kind++)
            for (int h = sub + chunk * RPW; h < a.heads[kind]; h += a.chunks * RPW) {
                uint8_t* out = a.dst[kind] + (int64_t)i * a.dnb1[kind] + (int64_t)h * a.dnb2[kind] + (int64_t)s * a.dnb3[kind];
                if (8 * l < a.hd) store_out8<V16>(out + 8 * l * (a.out_f32 ? 4 : 2), zero, a.out_f32);
            }
        return;
    }

    // HALVES: pair j of the lane turns by (cs[j], sn[j]); else value j is y * cs[j] + partner * sn[j]
    float cs[8], sn[8];
    if (lo < groups[0] + groups[1]) {
        if constexpr (HALVES) {
#pragma unroll
            for (int j = 0; j < 4; j++) angle_of(s_turns[c + j], p, cs[j], sn[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = c + j;
                cs[j] = 1.0f, sn[j] = 0.0f;
                if (e >= a.n_dims) continue;
                if (a.neox || !(j & 1)) angle_of(s_turns[a.neox ? (e < half ? e : e - half) : e >> 1], p, cs[j], sn[j]);
                else cs[j] = cs[j - 1], sn[j] = -sn[j - 1];   // (the pair's first value has -sin)
                if (a.neox ? e < half : !(j & 1)) sn[j] = -sn[j];
            }
        }
    }
    const int partner = !HALVES && a.neox ? (c < half ? lane + half / 8 : lane - half / 8) & 31 : lane;

    int first = 0;
    auto rows = [&](auto kind_) {
        constexpr int kind = decltype(kind_)::value;
        constexpr bool kTurn = kind < 2, kApart = HALVES && kTurn;   // (v's rows are not rotated: eight consecutive values per lane, one block's arithmetic instead of two)
        constexpr bool kTensor = CACHE == B200_TYPE_F32 || kind == 0;
        const int g_lo = max(lo, first) - first, g_hi = min(hi, first + groups[kind]) - first;
        first += groups[kind];
        if (g_lo >= g_hi) return;
        const bool normed = kTurn && a.w[kTurn ? kind : 0] != nullptr;
        float w[8];
        if (normed) {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = inside ? load_global(a.w[kTurn ? kind : 0] + (HALVES && j >= 4 ? a.hd / 2 - 4 : 0) + c + j) : 0.0f;
        }
        const int at = kApart ? c : 8 * l, last = a.heads[kind] - 1;
        const uint8_t* src = a.src[kind] + (int64_t)i * a.snb1[kind] + (int64_t)s * a.snb3[kind] + (inside ? at : 0) * ES;
        uint8_t* dst = a.dst[kind] + (int64_t)s * a.dnb3[kind] + (kTensor ? (int64_t)i : p) * a.dnb1[kind];
        const int64_t src_step = a.snb2[kind], dst_step = a.dnb2[kind];
        for (int g0 = g_lo; g0 < g_hi; g0 += U) {
            float f[U][8];
#pragma unroll
            for (int u = 0; u < U; u++) {   // lanes behind the last head take its row once more and store nothing
                const uint8_t* row = src + min((g0 + u) * RPW + sub, last) * src_step;
                if constexpr (kApart) load_in4x2<F32>(row, row + a.hd / 2 * ES, f[u]);
                else load_in8<F32, V16>(row, f[u]);
            }
            // the rows of the next turn into L2 meanwhile
            if (g0 + U < g_hi && (at * ES & 127) == 0) {
#pragma unroll
                for (int u = U; u < 2 * U; u++) {
                    const uint8_t* row = src + min((g0 + u) * RPW + sub, last) * src_step;
                    prefetch_l2(row);
                    if constexpr (kApart) prefetch_l2(row + a.hd / 2 * ES);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (g0 + u >= g_hi) break;
                const int h = (g0 + u) * RPW + sub;
                if (normed) {
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; j++) sum = fmaf(f[u][j], f[u][j], sum);
                    if (!inside) sum = 0.0f;
#pragma unroll
                    for (int m = LPR / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
                    const float r = rsqrtf(fmaf(sum, a.inv_hd, a.eps));
#pragma unroll
                    for (int j = 0; j < 8; j++) f[u][j] = f[u][j] * r * w[j];
                }
                if constexpr (kApart) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float x = f[u][j], y = f[u][4 + j];
                        f[u][j] = fmaf(x, cs[j], -y * sn[j]), f[u][4 + j] = fmaf(y, cs[j], x * sn[j]);
                    }
                } else if constexpr (kTurn) {
                    float other[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) other[j] = a.neox ? __shfl_sync(0xffffffffu, f[u][j], partner) : f[u][j ^ 1];
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (c + j < a.n_dims) f[u][j] = fmaf(f[u][j], cs[j], other[j] * sn[j]);
                }
                const bool live = h <= last && inside;
                uint8_t* out = dst + h * dst_step;
                if constexpr (kTensor) {
                    if (!live) continue;
                    if constexpr (HALVES) store_out4x2(out, c, f[u], a.hd, a.out_f32);
                    else store_out8<V16>(out + c * (a.out_f32 ? 4 : 2), f[u], a.out_f32);
                } else if constexpr (kApart) {
                    store_row4x2<CACHE>(out, l, f[u], live && stored, a.hd);
                } else {
                    store_row8<CACHE>(out, 8 * l, f[u], live && stored, a.hd);
                }
            }
        }
    };
    rows(std::integral_constant<int, 0>());
    rows(std::integral_constant<int, 1>());
    if constexpr (CACHE != B200_TYPE_F32) rows(std::integral_constant<int, 2>());
}

template <bool F32, bool V16, int CACHE>
cudaError_t launch_lanes(const RopeArgs& a, unsigned grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(32 * kRopeWarps);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if constexpr (V16) {
        if (a.neox && a.n_dims == a.hd && a.hd == 64) return cudaLaunchKernelEx(&cfg, qk_rope_kernel<F32, true, 8, CACHE, true>, a);
        if (a.neox && a.n_dims == a.hd && a.hd == 128) return cudaLaunchKernelEx(&cfg, qk_rope_kernel<F32, true, 16, CACHE, true>, a);
    }
    if (a.hd <= 32) return cudaLaunchKernelEx(&cfg, qk_rope_kernel<F32, V16, 4, CACHE, false>, a);
    if (a.hd <= 64) return cudaLaunchKernelEx(&cfg, qk_rope_kernel<F32, V16, 8, CACHE, false>, a);
    return cudaLaunchKernelEx(&cfg, qk_rope_kernel<F32, V16, 16, CACHE, false>, a);
}

template <int CACHE>
cudaError_t launch_rope(RopeArgs a, bool f32, bool v16, cudaStream_t st) {
    const int rpw = 32 / (a.hd <= 32 ? 4 : (a.hd <= 64 ? 8 : 16));
    int groups = 0;
    for (int x = 0; x < 3; x++) groups += (a.heads[x] + rpw - 1) / rpw;
    // Few tokens: a warp per group of rows.  Many: all of a token's rows in one warp, so that its angles are worked out once.
    const int64_t want = (148 * 16 + a.n_tokens - 1) / a.n_tokens;
    a.chunks = (int)(want < groups ? want : groups);
    const int64_t grid = ((int64_t)a.n_tokens * a.chunks + kRopeWarps - 1) / kRopeWarps;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    if (f32) return v16 ? launch_lanes<true, true, CACHE>(a, (unsigned)grid, st) : launch_lanes<true, false, CACHE>(a, (unsigned)grid, st);
    return v16 ? launch_lanes<false, true, CACHE>(a, (unsigned)grid, st) : launch_lanes<false, false, CACHE>(a, (unsigned)grid, st);
}

// Turns of the pairs per position as fractions of 2^64, in 80-bit arithmetic; a thread keeps the last parameters' table.
void fill_turns(const b200_rope_params& r, uint64_t (&out)[kMaxHalf]) {
    struct Table {
        float base = 0.0f, scale = 0.0f;
        int32_t n = 0;
        uint64_t turns[kMaxHalf] = {};
    };
    static thread_local Table t;
    if (t.n != r.n_dims || t.base != r.freq_base || t.scale != r.freq_scale) {
        const long double two_pi = 6.283185307179586476925286766559005768L;
        for (int i = 0; i < r.n_dims / 2; i++) {
            long double f = (long double)r.freq_scale / two_pi * powl((long double)r.freq_base, -2.0L * i / r.n_dims);
            f -= floorl(f);
            t.turns[i] = f < 1.0L ? (uint64_t)(f * 18446744073709551616.0L) : 0;   // (a tiny negative turn plus one rounds to a whole one)
        }
        t.n = r.n_dims, t.base = r.freq_base, t.scale = r.freq_scale;
    }
    memcpy(out, t.turns, sizeof(out));
}

struct Alignment {
    bool v16 = true;
    int check(const b200_tensor* t, int type_a, int type_b) {
        if (!t->data) return B200_E_NULL;
        if (t->type != type_a && t->type != type_b) return B200_E_TYPE;
        const uint64_t es = t->type == B200_TYPE_F32 ? 4 : 2;
        if (t->nb[0] != es || t->nb[1] % es || t->nb[2] % es || t->nb[3] % es) return B200_E_STRIDE;
        if ((uintptr_t)t->data % es) return B200_E_ALIGN;
        for (int i = 0; i < 4; i++)
            if (t->ne[i] <= 0) return B200_E_SHAPE;
        v16 = v16 && (uintptr_t)t->data % 16 == 0 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && t->nb[3] % 16 == 0;
        return B200_OK;
    }
};

void set_src(RopeArgs& a, int x, const b200_tensor* t) {
    a.src[x] = (const uint8_t*)t->data;
    a.snb1[x] = (int64_t)t->nb[1], a.snb2[x] = (int64_t)t->nb[2], a.snb3[x] = (int64_t)t->nb[3];
    a.heads[x] = (int)t->ne[2];
}
void set_dst(RopeArgs& a, int x, const b200_tensor* t) {
    a.dst[x] = (uint8_t*)t->data;
    a.dnb1[x] = (int64_t)t->nb[1], a.dnb2[x] = (int64_t)t->nb[2], a.dnb3[x] = (int64_t)t->nb[3];
}

// The parameters and norm weights of a call over rows of `hd` values.
int set_params(RopeArgs& a, int64_t hd, const b200_rope_params* r, const b200_tensor* const (&norm)[2]) {
    if (!r) return B200_E_NULL;
    if (hd <= 0 || hd % 8 || hd > 128) return B200_E_UNSUPPORTED;
    if (r->mode != B200_ROPE_NORM && r->mode != B200_ROPE_NEOX) return B200_E_UNSUPPORTED;
    if (r->n_dims < 0 || r->n_dims % 2 || r->n_dims > hd) return B200_E_SHAPE;
    if (r->mode == B200_ROPE_NEOX && r->n_dims % 16) return B200_E_UNSUPPORTED;   // a pair's two values in the same place of two lanes
    if (!std::isfinite(r->freq_base) || r->freq_base <= 0.0f || !std::isfinite(r->freq_scale) || !std::isfinite(r->eps) || r->eps < 0.0f) return B200_E_SHAPE;
    for (int x = 0; x < 2; x++) {
        const b200_tensor* w = norm[x];
        if (!w) continue;
        if (!w->data) return B200_E_NULL;
        if (w->type != B200_TYPE_F32) return B200_E_TYPE;
        if (w->ne[0] != hd || w->ne[1] != 1 || w->ne[2] != 1 || w->ne[3] != 1) return B200_E_SHAPE;
        if (w->nb[0] != 4) return B200_E_STRIDE;
        if ((uintptr_t)w->data % 4) return B200_E_ALIGN;
        a.w[x] = (const float*)w->data;
    }
    a.hd = (int)hd, a.n_dims = r->n_dims, a.neox = r->mode == B200_ROPE_NEOX, a.eps = r->eps, a.inv_hd = 1.0f / (float)hd;
    fill_turns(*r, a.turns);
    return B200_OK;
}

bool same_shape(const b200_tensor* x, const b200_tensor* y) {
    return x->ne[0] == y->ne[0] && x->ne[1] == y->ne[1] && x->ne[2] == y->ne[2] && x->ne[3] == y->ne[3];
}

int set_tokens(RopeArgs& a, int64_t n, int64_t streams) {
    if (n > INT32_MAX / 2 || streams > INT32_MAX / 2 || n * streams > INT32_MAX / 2) return B200_E_LIMIT;
    a.n = (int)n, a.n_tokens = (int)(n * streams);
    return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

B200_API int b200_qk_norm_rope(const b200_tensor* q, const b200_tensor* k, const b200_tensor* q_norm, const b200_tensor* k_norm,
                               const b200_rope_params* params, const int32_t* pos, int32_t pos0, const int32_t* n_rows, const b200_tensor* q_out,
                               const b200_tensor* k_out, void* cuda_stream) {
    if (!q || !q_out || (k == nullptr) != (k_out == nullptr)) return B200_E_NULL;
    RopeArgs a = {};
    Alignment al;
    int rc;
    const b200_tensor *in[2] = {q, k}, *out[2] = {q_out, k_out};
    for (int x = 0; x < (k ? 2 : 1); x++) {
        if ((rc = al.check(in[x], x ? q->type : B200_TYPE_F32, x ? q->type : B200_TYPE_F16))) return rc;
        if ((rc = al.check(out[x], x ? q_out->type : B200_TYPE_F32, x ? q_out->type : B200_TYPE_F16))) return rc;
        if (!same_shape(in[x], out[x]) || in[x]->ne[2] > 65535) return B200_E_SHAPE;
        set_src(a, x, in[x]), set_dst(a, x, out[x]);
    }
    if (k && (k->ne[0] != q->ne[0] || k->ne[1] != q->ne[1] || k->ne[3] != q->ne[3])) return B200_E_SHAPE;
    if ((rc = set_tokens(a, q->ne[1], q->ne[3]))) return rc;
    if ((rc = set_params(a, q->ne[0], params, {q_norm, k_norm}))) return rc;
    a.out_f32 = q_out->type == B200_TYPE_F32, a.pos = pos, a.pos0 = pos0, a.n_rows = n_rows;
    const cudaError_t e = launch_rope<B200_TYPE_F32>(a, q->type == B200_TYPE_F32, al.v16, (cudaStream_t)cuda_stream);
    if (e != cudaSuccess || cudaGetLastError() != cudaSuccess) return B200_E_CUDA;
    return B200_OK;
}

B200_API int b200_kv_append_rope(b200_kv_cache* kv, int layer, const b200_tensor* q, const b200_tensor* k_new, const b200_tensor* v_new,
                                 const b200_tensor* q_norm, const b200_tensor* k_norm, const b200_rope_params* params, const int32_t* pos, int32_t pos0,
                                 const int32_t* n_rows, const b200_tensor* q_out, void* cuda_stream) {
    if (!kv || !k_new || !v_new || (q == nullptr) != (q_out == nullptr)) return B200_E_NULL;
    if (layer < 0 || layer >= kv->cfg.n_layers) return B200_E_SHAPE;
    if (!on_current_device(kv)) return B200_E_STATE;
    RopeArgs a = {};
    Alignment al;
    int rc;
    b200_tensor view[2];
    b200_kv_view(kv, layer, kv->ctx_rows, &view[0], &view[1]);
    for (int x = 0; x < 2; x++) {
        const b200_tensor* t = x ? v_new : k_new;
        if ((rc = al.check(t, x ? k_new->type : B200_TYPE_F32, x ? k_new->type : B200_TYPE_F16))) return rc;
        if (t->ne[0] != kv->cfg.head_dim || t->ne[2] != kv->cfg.n_kv_heads || t->ne[3] != kv->cfg.n_streams) return B200_E_SHAPE;
        if (t->ne[1] != k_new->ne[1] || t->ne[1] > kv->ctx_rows) return B200_E_SHAPE;
        set_src(a, 1 + x, t), set_dst(a, 1 + x, &view[x]);
    }
    if (!pos && (pos0 < 0 || pos0 + k_new->ne[1] > kv->ctx_rows)) return B200_E_SHAPE;
    if (q) {
        if ((rc = al.check(q, k_new->type, k_new->type)) || (rc = al.check(q_out, B200_TYPE_F32, B200_TYPE_F16))) return rc;
        if (!same_shape(q, q_out) || q->ne[0] != k_new->ne[0] || q->ne[1] != k_new->ne[1] || q->ne[3] != k_new->ne[3] || q->ne[2] > 65535) return B200_E_SHAPE;
        set_src(a, 0, q), set_dst(a, 0, q_out);
        a.out_f32 = q_out->type == B200_TYPE_F32;
    }
    if ((rc = set_tokens(a, k_new->ne[1], k_new->ne[3]))) return rc;
    if ((rc = set_params(a, k_new->ne[0], params, {q_norm, k_norm}))) return rc;
    a.ctx_rows = (int)kv->ctx_rows, a.pos = pos, a.pos0 = pos0, a.n_rows = n_rows;
    const bool f32 = k_new->type == B200_TYPE_F32;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    cudaError_t e;
    switch (kv->cfg.type) {
        case B200_TYPE_F16: e = launch_rope<B200_TYPE_F16>(a, f32, al.v16, st); break;
        case B200_TYPE_Q8_0: e = launch_rope<B200_TYPE_Q8_0>(a, f32, al.v16, st); break;
        default: e = launch_rope<B200_TYPE_Q4_0>(a, f32, al.v16, st); break;
    }
    if (e != cudaSuccess || cudaGetLastError() != cudaSuccess) return B200_E_CUDA;
    return B200_OK;
}

}  // extern "C"
