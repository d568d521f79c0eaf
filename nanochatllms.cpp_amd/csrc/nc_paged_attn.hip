// nc_paged_attn.hip -- attention of requests' new rows over their pages of
// the K/V cache.
//
//   out[row, h] = sum_j softmax_j(q[row, h] . k[j, h / group] / sqrt(d)) v[j, h / group]
//
// over the positions j that the row sees: j <= p (p the row's own position),
// and with a window w > 0 also j > p - w or j < n_sink.
//
// The rows of a request that share a kv head, (token, head of the group)
// with the head fastest, are cut into tiles; a tile walks the positions in
// steps with a running maximum and sum of the softmax.  Scores are computed
// transposed, S^T = K Q^T: in the matrix cores' output layout a lane then
// holds scores of one query row, so the maximum, the sum and the rescaling
// are per-lane values, and the lane's own probabilities, packed to fp16, are
// already the operand that O^T = V^T P^T needs -- the positions behind the
// operand's slots are permuted alike for both factors, so nothing moves
// between lanes.
//
// Roundings: K, V and Q are fp16 (exact for fp16 tensors; a Q8 code times its
// delta rounds once, 2^-11 of the value, an eighth of a code's own step at
// full range), probabilities round to fp16 (2^-11 each; the fp16 result
// rounds as much), everything else is fp32.  Probabilities are scaled by 2^14
// so that what falls under fp16's smallest number is below 2^-38 of the
// maximum's weight.
#include "nc_act.h"
#include "nc_paged.h"

namespace nc {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float kPScale = 14.0f;  // log2 of the probabilities' scale

struct AttnArgs {
    const uint8_t* q;
    uint8_t* out;
    int q_pitch, out_pitch, q_dtype, out_dtype;
    const uint8_t *k, *v;
    const uint16_t *kd, *vd;
    const int *table, *row_start, *kv_len;
    int n_req, max_pages, n_pages, lps;
    int hq, hkv, group, max_tokens, max_new, max_kv;
    int window, sink;
    float scale;   // log2(e) / sqrt(d)
    int row_tiles; // tiles of a request, or tile slots in all
    int splits;    // parts of a tile's positions at most
    int part;      // steps of a part
    float* ws;     // [splits][max_tokens * hq][d] sums, then [splits][max_tokens * hq][2] (maximum, sum)
};

// The positions that a tile of rows visits, in steps of S: [0, n_sink) and
// [lo, hi), as one list of step numbers.
template <int S>
struct Steps {
    int sinks, first, count;
    __device__ __forceinline__ Steps(int lo, int hi, int sink)
    {
        first = lo / S;
        sinks = min((sink + S - 1) / S, first);
        count = sinks + (hi + S - 1) / S - first;
    }
    __device__ __forceinline__ int at(int v) const { return v < sinks ? v : first + v - sinks; }
};

// Rows [row0, row0 + M) of the request's (token, head) rows.
struct Tile {
    int n_rows;         // rows of the request
    int first_row;      // the request's first row of the tensors
    int row0;           // the tile's first (token, head) row
    int pos0;           // position of the request's first row
    int kv;             // positions cached
    int tok_lo, tok_hi; // the tile's tokens
    int lo, hi;         // visible positions [lo, hi) besides the sinks
};

template <int M>
__device__ __forceinline__ bool tile_of(const AttnArgs& a, int req, int row0, Tile& t)
{
    const RowSpan s = request_rows(a.row_start, req, a.max_tokens, 0x7FFFFFFF);
    const int kv = a.kv_len[req];
    const int limit = (int)min((long long)a.max_pages << a.lps, (long long)a.max_kv);
    if (kv > limit || kv < s.n) return false;  // lengths beyond the bounds: the rows are left as they were
    t.n_rows = min(s.n, a.max_new) * a.group;
    t.first_row = s.first;
    t.row0 = row0;
    t.kv = kv;
    t.pos0 = kv - s.n;
    if (row0 >= t.n_rows) return false;
    t.tok_lo = row0 / a.group;
    t.tok_hi = min(row0 + M, t.n_rows) - 1;
    t.tok_hi /= a.group;
    t.lo = a.window ? max(0, t.pos0 + t.tok_lo - a.window + 1) : 0;
    t.hi = t.pos0 + t.tok_hi + 1;
    return true;
}

// A page id, or -1 for an entry that is none: callers read page 0 in its
// place and take its positions for unseen.
__device__ __forceinline__ int page_at(const AttnArgs& a, int req, int pos)
{
    const int id = a.table[(size_t)req * a.max_pages + min(pos >> a.lps, a.max_pages - 1)];
    return (unsigned)id < (unsigned)a.n_pages ? id : -1;
}

// Four fp16 pairs of eight codes times a delta: a code plus 128 in the low
// bits of 0x6400 is the fp16 number 1152 + code, so the subtraction is exact
// and the product rounds once.
__device__ __forceinline__ half8 dequant8(uint2 c, uint16_t delta)
{
    const half2v bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const _Float16 d = __builtin_bit_cast(_Float16, delta);
    const half2v d2 = {d, d};
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = (i < 2 ? c.x : c.y) ^ 0x80808080u;
        const uint32_t p = __builtin_amdgcn_perm(0x64646464u, w, i & 1 ? 0x04030402u : 0x04010400u);
        out[i] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(half2v, p) + bias) * d2);
    }
    return __builtin_bit_cast(half8, out);
}


// Four of them.
__device__ __forceinline__ uint2 dequant4(uint32_t c, uint16_t delta)
{
    const half8 h = dequant8(make_uint2(c, 0), delta);
    const u32x4 w = __builtin_bit_cast(u32x4, h);
    return make_uint2(w.x, w.y);
}

// Eight values, from col on, of a q row as fp16.
__device__ __forceinline__ half8 q_values(const AttnArgs& a, const uint8_t* row, int col, int cols)
{
    if (a.q_dtype == F16) return *reinterpret_cast<const half8*>(row + 2 * col);
    return dequant8(*reinterpret_cast<const uint2*>(row + col),
                    reinterpret_cast<const uint16_t*>(row + cols)[col >> 5]);
}

// Eight results of one (row, head), from column c8 * 8 of the head on.
template <int D>
__device__ __forceinline__ void store_out(const AttnArgs& a, int row, int head, int c8, float (&v)[8])
{
    uint8_t* p = a.out + (size_t)row * a.out_pitch;
    if (a.out_dtype == F16) act_store8<F16>(p, head * (D / 8) + c8, 0, v);
    else act_store8<Q8>(p, head * (D / 8) + c8, a.hq * D, v);
}

__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---- sixteen rows a tile ------------------------------------------------------
//
// One workgroup of four wavefronts per (tile, kv head, part of the
// positions); each wavefront takes every fourth step of 32 positions, so a
// step's K and V go from memory to the registers of the one wavefront that
// uses them, with no shared memory and no barrier before the four results are
// joined.  K: lane l holds position l % 16 (of each half of the step), values
// from 8 (l / 16) on: the matrix operand as it is loaded.  V: a lane loads
// d / 16 neighbouring values of the eight positions that its probabilities
// belong to, one load per position with whole rows across sixteen lanes, and
// v_perm turns the 8 x d / 16 block into d / 16 operands in registers.

template <int D, int CDT>
struct Kv16 {
    static constexpr int kKs = D / 32;
    u32x4 k[2][CDT == Q8 ? kKs / 2 : kKs];
    uint32_t v[8][CDT == Q8 ? D / 64 : D / 32];
    uint16_t kd[2][CDT == Q8 ? kKs / 2 : 1], vd[CDT == Q8 ? 8 : 1];
    int page[2];

    // First of the eight values that lane group g holds of operand ks.
    static __device__ __forceinline__ int col(int ks, int g)
    {
        return CDT == Q8 ? (ks >> 1) * 64 + g * 16 + (ks & 1) * 8 : ks * 32 + g * 8;
    }

    __device__ __forceinline__ void load(const AttnArgs& a, int head, int pos, int p0, int p1, int c, int g)
    {
        page[0] = p0;
        page[1] = p1;
        const int mask = (1 << a.lps) - 1;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // row of the half step's first position
            const size_t row = ((((size_t)max(page[h], 0) * a.hkv + head) << a.lps) + ((pos + 16 * h) & mask));
            const size_t kr = row + c;
            if constexpr (CDT == Q8) {
#pragma unroll
                for (int i = 0; i < kKs / 2; i++) {
                    k[h][i] = *reinterpret_cast<const u32x4*>(a.k + kr * D + i * 64 + g * 16);
                    kd[h][i] = a.kd[kr * (D / 32) + i * 2 + (g >> 1)];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kKs; i++)
                    k[h][i] = *reinterpret_cast<const u32x4*>(a.k + (kr * D + i * 32 + g * 8) * 2);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const size_t vr = row + 4 * g + j;
                uint32_t* to = v[4 * h + j];
                if constexpr (CDT == Q8) {
                    const uint8_t* p = a.v + vr * D + c * (D / 16);
                    if constexpr (D == 128) {
                        const uint2 w = *reinterpret_cast<const uint2*>(p);
                        to[0] = w.x;
                        to[1] = w.y;
                    } else {
                        to[0] = *reinterpret_cast<const uint32_t*>(p);
                    }
                    vd[4 * h + j] = a.vd[vr * (D / 32) + c / (512 / D)];
                } else {
                    const uint8_t* p = a.v + (vr * D + c * (D / 16)) * 2;
                    if constexpr (D == 128) {
                        const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                        for (int i = 0; i < 4; i++) to[i] = w[i];
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(p);
                        to[0] = w.x;
                        to[1] = w.y;
                    }
                }
            }
        }
    }

    __device__ __forceinline__ half8 k_operand(int h, int ks) const
    {
        if constexpr (CDT == Q8) {
            const u32x4 w = k[h][ks >> 1];
            return dequant8(ks & 1 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), kd[h][ks >> 1]);
        } else {
            return __builtin_bit_cast(half8, k[h][ks]);
        }
    }

    // The fp16 values of V, D / 32 pairs per position.
    __device__ __forceinline__ void v_values(uint32_t (&w)[8][D / 32]) const
    {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (CDT == F16) {
#pragma unroll
                for (int i = 0; i < D / 32; i++) w[j][i] = v[j][i];
            } else if constexpr (D == 128) {
                const u32x4 x = __builtin_bit_cast(u32x4, dequant8(make_uint2(v[j][0], v[j][1]), vd[j]));
#pragma unroll
                for (int i = 0; i < 4; i++) w[j][i] = x[i];
            } else {
                const uint2 x = dequant4(v[j][0], vd[j]);
                w[j][0] = x.x;
                w[j][1] = x.y;
            }
        }
    }
};

__device__ __forceinline__ bool pair_not_finite(uint32_t w)
{
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}

// Operand dt of V^T: value dt of the eight positions.
template <int D>
__device__ __forceinline__ half8 v_operand(const uint32_t (&w)[8][D / 32], int dt)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = __builtin_amdgcn_perm(w[2 * i + 1][dt >> 1], w[2 * i][dt >> 1], dt & 1 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(half8, o);
}

template <int D, int CDT>
__global__ __launch_bounds__(256, 2) void k_paged_attn16(AttnArgs a)
{
    constexpr int kKs = D / 32, kDt = D / 16, kPitch = D + 4;
    __shared__ float o_sh[4][16][kPitch];
    __shared__ float ml_sh[4][16][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    int b = blockIdx.x;
    const int part = b % a.splits;
    b /= a.splits;
    const int head = b % a.hkv;
    b /= a.hkv;
    const int req = b / a.row_tiles;
    Tile t;
    if (!tile_of<16>(a, req, (b % a.row_tiles) * 16, t)) return;
    const Steps<32> steps(t.lo, t.hi, a.window ? a.sink : 0);
    const int v0 = part * a.part;
    if (v0 >= steps.count) return;
    const int v1 = part == a.splits - 1 ? steps.count : min(v0 + a.part, steps.count);
    const int parts = min((steps.count + a.part - 1) / a.part, a.splits);

    // this lane's row: q operand and position
    const int my = min(t.row0 + c, t.n_rows - 1);
    const int my_tok = my / a.group, my_pos = t.pos0 + my_tok;
    half8 q[kKs];
    {
        const uint8_t* row = a.q + (size_t)(t.first_row + my_tok) * a.q_pitch;
        const int col = (head * a.group + my % a.group) * D;
#pragma unroll
        for (int ks = 0; ks < kKs; ks++) q[ks] = q_values(a, row, col + Kv16<D, CDT>::col(ks, g), a.hq * D);
    }
    float m = -__builtin_inff(), sum = 0.0f;
    f32x4 o[kDt];
#pragma unroll
    for (int i = 0; i < kDt; i++) o[i] = f32x4{0, 0, 0, 0};

    auto fetch = [&](Kv16<D, CDT>& kv, int v) {
        const int pos = steps.at(v) * 32;
        kv.load(a, head, pos, page_at(a, req, pos), page_at(a, req, pos + 16), c, g);
    };
    auto use = [&](const Kv16<D, CDT>& kv, int v) {
        const int pos = steps.at(v) * 32;
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int ks = 0; ks < kKs; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) s[h] = mfma16(kv.k_operand(h, ks), q[ks], s[h]);
        const int last = t.pos0 + t.tok_hi;
        const bool all = pos + 31 <= t.pos0 + t.tok_lo && kv.page[0] >= 0 && kv.page[1] >= 0 &&
                         (!a.window || pos > last - a.window || pos + 31 < a.sink);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * a.scale;
        if (!all) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool seen = key <= my_pos && (!a.window || key > my_pos - a.window || key < a.sink) &&
                                  kv.page[j >> 2] >= 0;
                if (!seen) x[j] = -__builtin_inff();
            }
        }
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) mx = fmaxf(mx, x[j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(m, mx);
        const float base = m_new == -__builtin_inff() ? 0.0f : m_new - kPScale;
        const float alpha = __builtin_amdgcn_exp2f(m - kPScale - base);
        half8 p;
        float add = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float e = __builtin_amdgcn_exp2f(x[j] - base);
            add += e;
            p[j] = (_Float16)e;
        }
        sum = __builtin_fmaf(sum, alpha, add);
        m = m_new;
        if (__ballot(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < kDt; i++) o[i] *= alpha;
        }
        uint32_t w[8][D / 32];
        kv.v_values(w);
        bool odd = false;  // a value that no probability of 0 can hide
        if (!all) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool seen = key < t.hi && (!a.window || key >= t.lo || key < a.sink) && kv.page[j >> 2] >= 0;
#pragma unroll
                for (int i = 0; i < D / 32; i++) {
                    if (!seen) w[j][i] = 0;
                    odd |= pair_not_finite(w[j][i]);
                }
            }
        }
        if (!all && t.tok_lo != t.tok_hi && __ballot(odd)) {
            // positions that some of the tile's rows see and others do not
            // hold infinities or NaN: one token after the other, with its
            // unseen positions' values cleared
            for (int tok = t.tok_lo; tok <= t.tok_hi; tok++) {
                const int at = t.pos0 + tok;
                uint32_t u[8][D / 32];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                    const bool seen = key <= at && (!a.window || key > at - a.window || key < a.sink);
#pragma unroll
                    for (int i = 0; i < D / 32; i++) u[j][i] = seen ? w[j][i] : 0;
                }
#pragma unroll
                for (int i = 0; i < kDt; i++) {
                    const f32x4 r = mfma16(v_operand<D>(u, i), p, o[i]);
                    if (my_tok == tok) o[i] = r;
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kDt; i++) o[i] = mfma16(v_operand<D>(w, i), p, o[i]);
    };

    // two steps' loads in flight
    {
        Kv16<D, CDT> x, y;
        int v = v0 + wave;
        if (v < v1) fetch(x, v);
        while (v < v1) {
            if (v + 4 < v1) fetch(y, v + 4);
            use(x, v);
            v += 4;
            if (v >= v1) break;
            if (v + 4 < v1) fetch(x, v + 4);
            use(y, v);
            v += 4;
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);

    // join the wavefronts: lane (c, g) holds row c, values (4 g + i) (d / 16) + dt
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int dt = 0; dt < kDt; dt++) o_sh[wave][c][(4 * g + i) * kDt + dt] = o[dt][i];
    if (g == 0) {
        ml_sh[wave][c][0] = m;
        ml_sh[wave][c][1] = sum;
    }
    __syncthreads();
    const int rr = tid / (D / 8), c8 = tid % (D / 8);
    if (rr >= 16 || t.row0 + rr >= t.n_rows) return;  // whole heads
    float mw[4], top = -__builtin_inff(), total = 0.0f, r[8] = {};
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, mw[w] = ml_sh[w][rr][0]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float f = mw[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mw[w] - top);
        total += f * ml_sh[w][rr][1];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] += f * o_sh[w][rr][c8 * 8 + i];
    }
    const int row = t.row0 + rr, tok = t.first_row + row / a.group, qh = head * a.group + row % a.group;
    if (parts == 1) {
        const float inv = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] *= inv;
        store_out<D>(a, tok, qh, c8, r);
        return;
    }
    const size_t rows = (size_t)a.max_tokens * a.hq, at = part * rows + (size_t)tok * a.hq + qh;
    float4* dst = reinterpret_cast<float4*>(a.ws + at * D + c8 * 8);
    dst[0] = make_float4(r[0], r[1], r[2], r[3]);
    dst[1] = make_float4(r[4], r[5], r[6], r[7]);
    if (c8 == 0) {
        float* ml = a.ws + a.splits * rows * D + at * 2;
        ml[0] = top;
        ml[1] = total;
    }
}

// The parts of a tile joined in their order.
template <int D>
__global__ __launch_bounds__(16 * D / 8) void k_paged_join(AttnArgs a)
{
    int b = blockIdx.x;
    const int head = b % a.hkv;
    b /= a.hkv;
    Tile t;
    if (!tile_of<16>(a, b / a.row_tiles, (b % a.row_tiles) * 16, t)) return;
    const Steps<32> steps(t.lo, t.hi, a.window ? a.sink : 0);
    const int parts = min((steps.count + a.part - 1) / a.part, a.splits);
    const int rr = threadIdx.x / (D / 8), c8 = threadIdx.x % (D / 8);
    if (parts <= 1 || t.row0 + rr >= t.n_rows) return;
    const int row = t.row0 + rr, tok = t.first_row + row / a.group, qh = head * a.group + row % a.group;
    const size_t rows = (size_t)a.max_tokens * a.hq, at = (size_t)tok * a.hq + qh;
    const float2* ml = reinterpret_cast<const float2*>(a.ws + a.splits * rows * D) + at;
    float top = -__builtin_inff(), total = 0.0f, r[8] = {};
    for (int s = 0; s < parts; s++) top = fmaxf(top, ml[s * rows].x);
    for (int s = 0; s < parts; s++) {
        const float2 e = ml[s * rows];
        const float f = e.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(e.x - top);
        total += f * e.y;
        const float4* src = reinterpret_cast<const float4*>(a.ws + (s * rows + at) * D + c8 * 8);
        const float4 u = src[0], w = src[1];
        r[0] += f * u.x;
        r[1] += f * u.y;
        r[2] += f * u.z;
        r[3] += f * u.w;
        r[4] += f * w.x;
        r[5] += f * w.y;
        r[6] += f * w.z;
        r[7] += f * w.w;
    }
    const float inv = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] *= inv;
    store_out<D>(a, tok, qh, c8, r);
}

// ---- launches -----------------------------------------------------------------

static void attn_shape(AttnArgs& a, int window, int n_sink)
{
    a.row_tiles = (int)(((long long)min(a.max_new, a.max_tokens) * a.group + 15) / 16);
    const long long tiles = (long long)a.n_req * a.row_tiles * a.hkv;
    // steps of a tile at most
    long long most = ((long long)a.max_kv + 31) / 32;
    if (window) {
        const long long seen = (n_sink + 31ll) / 32 + (window + 16ll) / 32 + 2;
        if (seen < most) most = seen;
    }
    if (most < 1) most = 1;
    long long want = tiles > 0 ? (1024 + tiles - 1) / tiles : 1;
    const long long cap = (most + 3) / 4;  // a step for each wavefront
    if (want > cap) want = cap;
    const long long by_len = (most + 31) / 32;  // 1024 positions
    if (want < by_len && tiles < 65536) want = by_len;
    if (want > 256) want = 256;
    a.part = (int)(((most + want - 1) / want + 3) / 4 * 4);
    a.splits = (int)((most + a.part - 1) / a.part);
}

static size_t attn_ws_bytes(const AttnArgs& a, int d)
{
    return a.splits > 1 ? (size_t)a.splits * a.max_tokens * a.hq * (d + 2) * 4 : 0;
}

static int attn_args(AttnArgs& a, const nc_paged_cache* cache, const nc_paged_batch* b, int n_heads, int window,
                     int n_sink)
{
    if (int s = check_cache("paged_attn", cache)) return s;
    if (int s = check_batch("paged_attn", b, cache->page_size)) return s;
    NC_CHECK_ARG(n_heads >= 1 && n_heads <= 1024 && n_heads % cache->n_kv_heads == 0,
                 "paged_attn: %d heads over %d kv heads", n_heads, cache->n_kv_heads);
    NC_CHECK_ARG(window >= 0 && n_sink >= 0, "paged_attn: window %d, sinks %d", window, n_sink);
    a.k = (const uint8_t*)cache->k;
    a.v = (const uint8_t*)cache->v;
    a.kd = (const uint16_t*)cache->k_deltas;
    a.vd = (const uint16_t*)cache->v_deltas;
    a.table = b->block_table;
    a.row_start = b->row_start;
    a.kv_len = b->kv_len;
    a.n_req = b->n_req;
    a.max_pages = b->max_pages;
    a.n_pages = cache->n_pages;
    a.lps = __builtin_ctz((unsigned)cache->page_size);
    a.hq = n_heads;
    a.hkv = cache->n_kv_heads;
    a.group = n_heads / cache->n_kv_heads;
    a.max_tokens = b->max_tokens;
    a.max_new = b->max_new;
    a.max_kv = b->max_kv;
    a.window = window;
    a.sink = window ? (n_sink < a.max_kv ? n_sink : a.max_kv) : 0;
    a.scale = (float)(1.4426950408889634 / sqrt((double)cache->d_head));
    attn_shape(a, window, a.sink);
    return NC_OK;
}

template <int D, int CDT>
static int attn_launch(const AttnArgs& a, hipStream_t st)
{
    const long long tiles = (long long)a.n_req * a.row_tiles * a.hkv;
    NC_CHECK_ARG(tiles * a.splits * 256 <= 0x7FFFFFFFll * 2, "paged_attn: %lld tiles are too many", tiles);
    hipLaunchKernelGGL((k_paged_attn16<D, CDT>), dim3((unsigned)(tiles * a.splits)), dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((k_paged_join<D>), dim3((unsigned)tiles), dim3(16 * D / 8), 0, st, a);
    return launch_status("k_paged_attn16");
}

}  // namespace nc

using namespace nc;

extern "C" int nc_paged_attn_workspace(const nc_paged_cache* cache, const nc_paged_batch* b, int n_heads, int window,
                                       int n_sink, size_t* bytes)
{
    NC_CHECK_ARG(bytes, "paged_attn_workspace: null result");
    AttnArgs a{};
    if (int s = attn_args(a, cache, b, n_heads, window, n_sink)) return s;
    *bytes = attn_ws_bytes(a, cache->d_head);
    return NC_OK;
}

extern "C" int nc_paged_attn(const nc_tensor* q, const nc_paged_cache* cache, const nc_paged_batch* b, nc_tensor* out,
                             int n_heads, int window, int n_sink, void* workspace, size_t workspace_bytes,
                             void* stream)
{
    AttnArgs a{};
    if (int s = attn_args(a, cache, b, n_heads, window, n_sink)) return s;
    const int cols = n_heads * cache->d_head;
    NC_CHECK_ARG(paged_rows_ok(q, b->max_tokens, cols) && paged_rows_ok(out, b->max_tokens, cols),
                 "paged_attn: q and out are not %d aligned rows of %d values", b->max_tokens, cols);
    NC_CHECK_ARG((q->dtype == NC_F16 || q->dtype == NC_Q8) && (out->dtype == NC_F16 || out->dtype == NC_Q8),
                 "paged_attn: dtypes %d, %d (F16 or Q8)", q->dtype, out->dtype);
    const size_t need = attn_ws_bytes(a, cache->d_head);
    NC_CHECK_ARG(need <= workspace_bytes && (!need || (workspace && aligned16(workspace))),
                 "paged_attn: workspace of %zu bytes (needs %zu, 16-byte aligned)", workspace_bytes, need);
    if (b->max_tokens == 0 || b->max_new == 0 || b->max_kv == 0) return NC_OK;
    a.q = (const uint8_t*)q->data;
    a.q_pitch = q->pitch;
    a.q_dtype = q->dtype;
    a.out = (uint8_t*)out->data;
    a.out_pitch = out->pitch;
    a.out_dtype = out->dtype;
    a.ws = (float*)workspace;
    hipStream_t st = stream_of(stream);
    if (cache->dtype == NC_Q8) return cache->d_head == 64 ? attn_launch<64, Q8>(a, st) : attn_launch<128, Q8>(a, st);
    return cache->d_head == 64 ? attn_launch<64, F16>(a, st) : attn_launch<128, F16>(a, st);
}
