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
// Roundings: K, V and Q are fp16, probabilities round to fp16 (2^-11 each;
// the fp16 result rounds as much), everything else is fp32.  Probabilities are scaled by 2^14
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

// Four codes as fp16 numbers: a code plus 128 in the low bits of 0x6400 is
// the fp16 number 1152 + code, so the subtraction is exact.
__device__ __forceinline__ void codes4(uint32_t c, half2v (&v)[2])
{
    const half2v bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t w = c ^ 0x80808080u;
    v[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias;
    v[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias;
}

// The products of eight codes and a delta in fp16, rounded once (hi), and
// what that rounding left (lo; hi + lo is the product, its 18 bits exactly).
struct HalfPair8 {
    half8 hi, lo;
};
__device__ __forceinline__ HalfPair8 dequant8(uint2 c, uint16_t delta)
{
    const _Float16 d = __builtin_bit_cast(_Float16, delta);
    const half2v d2 = {d, d};
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        half2v v[2];
        codes4(i ? c.y : c.x, v);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const half2v h = v[j] * d2;
            hi[2 * i + j] = __builtin_bit_cast(uint32_t, h);
            lo[2 * i + j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v[j], d2, -h));
        }
    }
    return {__builtin_bit_cast(half8, hi), __builtin_bit_cast(half8, lo)};
}

// Eight values, from col on, of a q row of `cols`.
template <int QDT>
__device__ __forceinline__ HalfPair8 q_values(const uint8_t* row, int col, int cols)
{
    if constexpr (QDT == F16) return {*reinterpret_cast<const half8*>(row + 2 * col), half8{}};
    else
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
// v_perm turns the 8 x d / 16 block into d / 16 operands in registers.  The
// next step's K is requested as soon as this step's is used up, and so its V:
// the same registers are always in flight or in use.
//
// A Q8 value is its code times its delta, 18 bits: here it enters as two
// fp16 halves, so a Q8 cache adds no rounding of its own.

__device__ __forceinline__ bool pair_not_finite(uint32_t w)
{
    return ((w & 0x7C00u) == 0x7C00u) | ((w & 0x7C000000u) == 0x7C000000u);
}

// Page, rows and lane offsets of one 32-position step.
template <int D, int CDT>
struct Kv16 {
    static constexpr int kKs = D / 32;
    static constexpr int kRow = CDT == Q8 ? D : 2 * D;  // bytes of a row
    static constexpr int kNk = CDT == Q8 ? kKs / 2 : kKs;
    static constexpr int kNv = CDT == Q8 ? D / 64 : D / 32;
    u32x4 k[2][kNk];
    uint32_t v[8][kNv];
    uint16_t kd[2][kNk], vd[8];

    // First of the eight values that lane group g holds of operand ks.
    static __device__ __forceinline__ int col(int ks, int g)
    {
        return CDT == Q8 ? (ks >> 1) * 64 + g * 16 + (ks & 1) * 8 : ks * 32 + g * 8;
    }

    // `row`: the cache row of the half step's first position.
    __device__ __forceinline__ void load_k(const AttnArgs& a, int h, size_t row, int c, int g)
    {
        const uint8_t* base = a.k + row * kRow;
        const uint32_t at = c * kRow + g * 16;
#pragma unroll
        for (int i = 0; i < kNk; i++) k[h][i] = *reinterpret_cast<const u32x4*>(base + (at + i * 64));
        if constexpr (CDT == Q8) {
            const uint16_t* db = a.kd + row * (D / 32);
            const uint32_t dat = c * (D / 32) + (g >> 1);
#pragma unroll
            for (int i = 0; i < kNk; i++) kd[h][i] = db[dat + 2 * i];
        }
    }

    __device__ __forceinline__ void load_v(const AttnArgs& a, int h, size_t row, int c, int g)
    {
        const uint8_t* base = a.v + row * kRow;
        const uint32_t at = 4 * g * kRow + c * (kRow / 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint8_t* p = base + (at + j * kRow);
            if constexpr (kNv == 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(p);
                v[4 * h + j][0] = w.x, v[4 * h + j][1] = w.y, v[4 * h + j][2] = w.z, v[4 * h + j][3] = w.w;
            } else if constexpr (kNv == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(p);
                v[4 * h + j][0] = w.x, v[4 * h + j][1] = w.y;
            } else {
                v[4 * h + j][0] = *reinterpret_cast<const uint32_t*>(p);
            }
        }
        if constexpr (CDT == Q8) {
            const uint16_t* db = a.vd + row * (D / 32);
            const uint32_t dat = 4 * g * (D / 32) + c / (512 / D);
#pragma unroll
            for (int j = 0; j < 4; j++) vd[4 * h + j] = db[dat + j * (D / 32)];
        }
    }

    __device__ __forceinline__ HalfPair8 k_operand(int h, int ks) const
    {
        if constexpr (CDT == Q8) {
            const u32x4 w = k[h][ks >> 1];
            return dequant8(ks & 1 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), kd[h][ks >> 1]);
        } else {
            return {__builtin_bit_cast(half8, k[h][ks]), half8{}};
        }
    }

    // Position j's values where `keep` has ones, zeros where it has none.
    __device__ __forceinline__ void v_clear(int j, uint32_t keep)
    {
#pragma unroll
        for (int i = 0; i < kNv; i++) v[j][i] &= keep;
        if constexpr (CDT == Q8) vd[j] &= (uint16_t)keep;
    }

    // Whether position j may hold an infinity or NaN.
    __device__ __forceinline__ bool v_not_finite(int j) const
    {
        if constexpr (CDT == Q8) return (vd[j] & 0x7FFFu) >= 0x6000u;  // a delta of 512: 128 of them pass fp16
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kNv; i++) odd |= pair_not_finite(v[j][i]);
        return odd;
    }

    // Pair i (values 2 i and 2 i + 1 of the lane's d / 16) of position j.
    __device__ __forceinline__ void v_pair(int j, int i, uint32_t& hi, uint32_t& lo) const
    {
        if constexpr (CDT == Q8) {
            const _Float16 d = __builtin_bit_cast(_Float16, vd[j]);
            const half2v d2 = {d, d};
            half2v x[2];
            codes4(v[j][i >> 1], x);
            const half2v h = x[i & 1] * d2;
            hi = __builtin_bit_cast(uint32_t, h);
            lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x[i & 1], d2, -h));
        } else {
            hi = v[j][i];
            lo = 0;
        }
    }
};

// Matrix operand of value 2 i + odd of eight positions, from their pairs i.
__device__ __forceinline__ half8 v_operand(const uint32_t (&w)[8], bool odd)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], odd ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(half8, o);
}

// MULTI: tiles may hold rows of several tokens, which see different positions.
// Single tokens have no use for what handles those, and its registers cost
// them a quarter of the wavefronts.
template <int D, int CDT, int QDT, bool MULTI>
__global__ __launch_bounds__(256, D == 64 && !MULTI ? 4 : (D == 64 || !MULTI ? 3 : 2)) void k_paged_attn16(AttnArgs a)
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
    const int my_tok = my / a.group, my_pos = t.pos0 + my_tok, my_lo = a.window ? my_pos - a.window + 1 : 0;
    HalfPair8 q[kKs];
    {
        const uint8_t* row = a.q + (size_t)(t.first_row + my_tok) * a.q_pitch;
        const int col = (head * a.group + my % a.group) * D;
#pragma unroll
        for (int ks = 0; ks < kKs; ks++)
            q[ks] = q_values<QDT>(row, col + Kv16<D, CDT>::col(ks, g), a.hq * D);
    }
    float m = -__builtin_inff(), sum = 0.0f;
    f32x4 o[kDt];
#pragma unroll
    for (int i = 0; i < kDt; i++) o[i] = f32x4{0, 0, 0, 0};

    Kv16<D, CDT> kv;
    const int mask = (1 << a.lps) - 1;
    auto row_of = [&](int page, int pos) {
        return (((size_t)max(page, 0) * a.hkv + head) << a.lps) + (pos & mask);
    };
    int v = v0 + wave;
    int pos = 0, p0 = 0, p1 = 0;
    if (v < v1) {
        pos = steps.at(v) * 32;
        p0 = page_at(a, req, pos);
        p1 = page_at(a, req, pos + 16);
        kv.load_k(a, 0, row_of(p0, pos), c, g);
        kv.load_k(a, 1, row_of(p1, pos + 16), c, g);
        kv.load_v(a, 0, row_of(p0, pos), c, g);
        kv.load_v(a, 1, row_of(p1, pos + 16), c, g);
    }
    while (v < v1) {
        const int nv = v + 4;
        int npos = 0, np0 = 0, np1 = 0;
        if (nv < v1) {
            npos = steps.at(nv) * 32;
            np0 = page_at(a, req, npos);
            np1 = page_at(a, req, npos + 16);
        }
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int ks = 0; ks < kKs; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const HalfPair8 k = kv.k_operand(h, ks);
                s[h] = mfma16(k.hi, q[ks].hi, s[h]);
                if constexpr (CDT == Q8) s[h] = mfma16(k.lo, q[ks].hi, s[h]);
                if constexpr (QDT == Q8) s[h] = mfma16(k.hi, q[ks].lo, s[h]);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (nv < v1) {
            kv.load_k(a, 0, row_of(np0, npos), c, g);
            kv.load_k(a, 1, row_of(np1, npos + 16), c, g);
        }
        const int last = t.pos0 + t.tok_hi;
        const bool all = pos + 31 <= t.pos0 + t.tok_lo && p0 >= 0 && p1 >= 0 &&
                         (!a.window || pos > last - a.window || pos + 31 < a.sink);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * a.scale;
        if (!all) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool seen = (key <= my_pos) & ((key >= my_lo) | (key < a.sink)) & ((j < 4 ? p0 : p1) >= 0);
                x[j] = seen ? x[j] : -__builtin_inff();
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
        // O^T += V^T P^T; positions that no row of the tile sees are cleared,
        // for a probability of 0 does not hide an infinity or NaN
        bool by_token = false;
        if (!all) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool seen = (key < t.hi) & ((key >= t.lo) | (key < a.sink)) & ((j < 4 ? p0 : p1) >= 0);
                kv.v_clear(j, seen ? ~0u : 0u);
            }
            if (MULTI && t.tok_lo != t.tok_hi) {
                bool odd = false;
#pragma unroll
                for (int j = 0; j < 8; j++) odd |= kv.v_not_finite(j);
                by_token = __ballot(odd) != 0;
            }
        }
        if (!by_token) {
#pragma unroll
            for (int i = 0; i < kDt / 2; i++) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j++) kv.v_pair(j, i, hi[j], lo[j]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    o[2 * i + e] = mfma16(v_operand(hi, e), p, o[2 * i + e]);
                    if constexpr (CDT == Q8) o[2 * i + e] = mfma16(v_operand(lo, e), p, o[2 * i + e]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // positions that some of the tile's rows see and others do not
            // hold infinities or NaN: one token after the other, with the
            // values of the positions that it does not see cleared
            for (int tok = t.tok_lo; tok <= t.tok_hi; tok++) {
                const int at = t.pos0 + tok, at_lo = a.window ? at - a.window + 1 : 0;
                uint32_t mine[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int key = pos + 16 * (j >> 2) + 4 * g + (j & 3);
                    mine[j] = (key <= at) & ((key >= at_lo) | (key < a.sink)) ? ~0u : 0u;
                }
#pragma unroll
                for (int i = 0; i < kDt / 2; i++) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        kv.v_pair(j, i, hi[j], lo[j]);
                        hi[j] &= mine[j];
                        lo[j] &= mine[j];
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        f32x4 r = mfma16(v_operand(hi, e), p, o[2 * i + e]);
                        if constexpr (CDT == Q8) r = mfma16(v_operand(lo, e), p, r);
                        if (my_tok == tok) o[2 * i + e] = r;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (nv < v1) {
            kv.load_v(a, 0, row_of(np0, npos), c, g);
            kv.load_v(a, 1, row_of(np1, npos + 16), c, g);
        }
        v = nv;
        pos = npos;
        p0 = np0;
        p1 = np1;
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
    const dim3 grid((unsigned)(tiles * a.splits));
    const bool multi = a.max_new > 1;
    if (a.q_dtype == F16) {
        if (multi) hipLaunchKernelGGL((k_paged_attn16<D, CDT, F16, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_paged_attn16<D, CDT, F16, false>), grid, dim3(256), 0, st, a);
    } else {
        if (multi) hipLaunchKernelGGL((k_paged_attn16<D, CDT, Q8, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_paged_attn16<D, CDT, Q8, false>), grid, dim3(256), 0, st, a);
    }
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
