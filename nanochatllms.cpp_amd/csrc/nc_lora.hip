// nc_lora.hip -- low-rank adapters of many requests beside a shared
// projection: out = base + scale (x a^T) b^T, each request with its own.
#include "nc_act.h"
#include "nc_paged.h"

namespace nc {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const uint8_t* x;
    const float* base;
    const uint16_t *a, *b;
    const float* scale;
    const int *adapter, *row_start;
    uint8_t* out;
    int x_pitch, base_pitch, out_pitch;
    int n_adapters, rank, k, n, n_req, max_tokens, max_new;
    int chunk;  // columns of a workgroup, a multiple of 128
};

// Eight ranks of a row of a or b from `at` on, zero past `rank`.
__device__ __forceinline__ half8 rank8(const uint16_t* row, int at, int rank)
{
    if ((rank & 7) == 0) {
        half8 z = {};
        return at < rank ? *reinterpret_cast<const half8*>(row + at) : z;
    }
    half8 v;
#pragma unroll
    for (int i = 0; i < 8; i++)
        v[i] = at + i < rank ? __builtin_bit_cast(_Float16, row[min(at + i, rank - 1)]) : (_Float16)0.0f;
    return v;
}

// One workgroup: sixteen rows of one request times `chunk` columns.  First
// the rows' low-rank products t = a x, as t^T = a x^T on the matrix cores
// with the four wavefronts taking every fourth 32 of k, summed in shared
// memory; then 32 columns at a time per wavefront, out^T = b t^T, the base
// added and the result stored by the lane that holds it.
//
// t has to enter the second product in fp16: it is split into a high and a
// low half (t = hi + lo to 2^-22 of the row's largest, after scaling the row
// by a power of two), so the product is as good as fp32 ones.  x's Q8 codes
// are exact in fp16 and a block's sum is multiplied by its delta in fp32.
template <int XDT, int ODT, int RT>
__global__ __launch_bounds__(256) void k_lora(LoraArgs a)
{
    constexpr int kR = RT * 16, kKs = (RT + 1) / 2, kTp = kKs * 32 + 4;
    __shared__ float part[4][16][kTp];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x;
    const int req = tile_request(a.row_start, a.n_req, tile, 1, 16, a.max_tokens);
    const RowSpan s = request_rows(a.row_start, req, a.max_tokens, a.max_new);
    const int row0 = (tile - first_tile(a.row_start[req], req, 1, 16, a.max_tokens)) * 16;
    if (row0 < 0 || row0 >= s.n) return;
    const int id = a.adapter[req];
    const bool some = (unsigned)id < (unsigned)a.n_adapters;
    const bool live = row0 + c < s.n;
    const int row = s.first + min(row0 + c, s.n - 1);

    float unit = 0.0f;
    half8 hi[kKs], lo[kKs];
    if (some) {
        const uint16_t* wa = a.a + (size_t)id * a.rank * a.k;
        const uint8_t* x = a.x + (size_t)row * a.x_pitch;
        f32x4 t[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) t[i] = f32x4{0, 0, 0, 0};
        const int steps = a.k / 32;
#pragma unroll 4
        for (int ks = wave; ks < steps; ks += 4) {
            half8 xv;
            float d = 1.0f;
            if constexpr (XDT == Q8) {
                const uint2 q = *reinterpret_cast<const uint2*>(x + ks * 32 + g * 8);
                d = h2f(reinterpret_cast<const uint16_t*>(x + a.k)[ks]);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    xv[i] = (_Float16)(float)(int8_t)((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xFFu);
            } else {
                xv = *reinterpret_cast<const half8*>(x + (ks * 32 + g * 8) * 2);
            }
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const int r = i * 16 + c;
                half8 av = {};
                if (r < a.rank) av = *reinterpret_cast<const half8*>(wa + (size_t)r * a.k + ks * 32 + g * 8);
                if constexpr (XDT == Q8) {
                    const f32x4 z = {0, 0, 0, 0};
                    const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, xv, z, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; j++) t[i][j] = __builtin_fmaf(p[j], d, t[i][j]);
                } else {
                    t[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, xv, t[i], 0, 0, 0);
                }
            }
        }
        // lane (c, g): row c, ranks 16 i + 4 g + j
#pragma unroll
        for (int i = 0; i < RT; i++)
            *reinterpret_cast<f32x4*>(&part[wave][c][i * 16 + 4 * g]) = t[i];
        if constexpr (RT & 1)
            *reinterpret_cast<f32x4*>(&part[wave][c][kR + 4 * g]) = f32x4{0, 0, 0, 0};
        __syncthreads();
        float v[kKs][8], top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKs; ks++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int r = ks * 32 + g * 8 + j;
                v[ks][j] = (part[0][c][r] + part[1][c][r]) + (part[2][c][r] + part[3][c][r]);
                top = fmaxf(top, fabsf(v[ks][j]));
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // the row's largest to [2^13, 2^14)
        const int e = top > 0.0f && top < __builtin_inff() ? 14 - (ilogbf(top) + 1) : 0;
        unit = ldexpf(a.scale[id], -e);
#pragma unroll
        for (int ks = 0; ks < kKs; ks++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float f = ldexpf(v[ks][j], e);
                hi[ks][j] = (_Float16)f;
                const float rest = f - (float)hi[ks][j];
                lo[ks][j] = (_Float16)(fabsf(f) < __builtin_inff() ? rest : 0.0f);
            }
    }
    const uint16_t* wb = a.b + (some ? (size_t)id * a.n * a.rank : 0);
    const int n0 = blockIdx.y * a.chunk, n1 = min(n0 + a.chunk, a.n);
    const bool vec = (a.n & 3) == 0;
    for (int n = n0 + wave * 32; n < n1; n += 128) {
        f32x4 y[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            y[u] = f32x4{0, 0, 0, 0};
            if (some) {
                const int col = min(n + u * 16 + c, a.n - 1);
#pragma unroll
                for (int ks = 0; ks < kKs; ks++) {
                    const half8 bv = rank8(wb + (size_t)col * a.rank, ks * 32 + g * 8, a.rank);
                    y[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv, hi[ks], y[u], 0, 0, 0);
                    y[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv, lo[ks], y[u], 0, 0, 0);
                }
            }
        }
        // lane (c, g): row c, columns n + 16 u + 4 g + j
        const float* bp = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.base) +
                                                         (size_t)row * a.base_pitch);
        uint8_t* op = a.out + (size_t)row * a.out_pitch;
        float r[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int col = n + u * 16 + 4 * g;
            float bv[4] = {};
            if (vec && col < n1) {
                const float4 w = *reinterpret_cast<const float4*>(bp + col);
                bv[0] = w.x, bv[1] = w.y, bv[2] = w.z, bv[3] = w.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (col + j < n1) bv[j] = bp[col + j];
            }
#pragma unroll
            for (int j = 0; j < 4; j++) r[u][j] = some ? __builtin_fmaf(y[u][j], unit, bv[j]) : bv[j];
        }
        if constexpr (ODT == Q8) {
            // the 32 columns are one block, on the lanes of the row
            float top = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (n + u * 16 + 4 * g + j < n1) top = fmaxf(top, fabsf(r[u][j]));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float delta = top / 127.0f;
            const float inv = delta != 0.0f ? 1.0f / delta : 0.0f;
            if (live) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int col = n + u * 16 + 4 * g;
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int8_t q = col + j < n1 ? (int8_t)roundf(r[u][j] * inv) : (int8_t)0;
                        w |= (uint32_t)(uint8_t)q << (8 * j);
                    }
                    *reinterpret_cast<uint32_t*>(op + col) = w;  // codes come in whole blocks
                }
                if (g == 0) reinterpret_cast<uint16_t*>(op + act_delta_offset(a.n))[n >> 5] = f2h(delta);
            }
        } else if (live) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int col = n + u * 16 + 4 * g;
                if (ODT == F32) {
                    float* o = reinterpret_cast<float*>(op) + col;
                    if (vec && col < n1) {
                        *reinterpret_cast<float4*>(o) = make_float4(r[u][0], r[u][1], r[u][2], r[u][3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (col + j < n1) o[j] = r[u][j];
                    }
                } else {
                    uint16_t* o = reinterpret_cast<uint16_t*>(op) + col;
                    if (vec && col < n1) {
                        *reinterpret_cast<uint2*>(o) =
                            make_uint2((uint32_t)f2h(r[u][0]) | (uint32_t)f2h(r[u][1]) << 16,
                                       (uint32_t)f2h(r[u][2]) | (uint32_t)f2h(r[u][3]) << 16);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (col + j < n1) o[j] = f2h(r[u][j]);
                    }
                }
            }
        }
    }
}

template <int XDT, int ODT>
static void lora_launch(const LoraArgs& a, dim3 grid, hipStream_t st)
{
    if (a.rank <= 16) hipLaunchKernelGGL((k_lora<XDT, ODT, 1>), grid, dim3(256), 0, st, a);
    else if (a.rank <= 32) hipLaunchKernelGGL((k_lora<XDT, ODT, 2>), grid, dim3(256), 0, st, a);
    else if (a.rank <= 64) hipLaunchKernelGGL((k_lora<XDT, ODT, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_lora<XDT, ODT, 8>), grid, dim3(256), 0, st, a);
}

}  // namespace nc

using namespace nc;

extern "C" int nc_lora_add(const nc_tensor* x, const nc_tensor* base, const nc_lora* lora, const int32_t* adapter,
                           const int32_t* row_start, int n_req, int max_new, nc_tensor* out, void* stream)
{
    NC_CHECK_ARG(lora && lora->a && lora->b && lora->scale && adapter && row_start, "lora_add: null argument");
    NC_CHECK_ARG(lora->rank >= 1 && lora->rank <= NC_LORA_MAX_RANK, "lora_add: rank %d (1 to %d)", lora->rank,
                 NC_LORA_MAX_RANK);
    NC_CHECK_ARG(lora->k >= 32 && lora->k % 32 == 0 && lora->n >= 1 && lora->n_adapters >= 1,
                 "lora_add: %d adapters [%d, %d] (k a multiple of 32)", lora->n_adapters, lora->n, lora->k);
    NC_CHECK_ARG(aligned16(lora->a) && aligned16(lora->b), "lora_add: adapters are not 16-byte aligned");
    NC_CHECK_ARG(n_req >= 1 && n_req <= NC_PAGED_MAX_REQ && max_new >= 0, "lora_add: %d requests of %d rows", n_req,
                 max_new);
    const int rows = x ? x->rows : 0;
    NC_CHECK_ARG(paged_rows_ok(x, 0, lora->k) && (x->dtype == NC_F16 || x->dtype == NC_Q8) && rows >= 0 &&
                     rows <= (1 << 26),
                 "lora_add: x is not aligned rows of %d values, F16 or Q8", lora->k);
    NC_CHECK_ARG(paged_rows_ok(base, rows, lora->n) && base->dtype == NC_F32,
                 "lora_add: base is not %d aligned fp32 rows of %d values", rows, lora->n);
    NC_CHECK_ARG(paged_rows_ok(out, rows, lora->n), "lora_add: out is not %d aligned rows of %d values", rows, lora->n);
    if (rows == 0 || max_new == 0) return NC_OK;
    LoraArgs a{};
    a.x = (const uint8_t*)x->data;
    a.x_pitch = x->pitch;
    a.base = (const float*)base->data;
    a.base_pitch = base->pitch;
    a.out = (uint8_t*)out->data;
    a.out_pitch = out->pitch;
    a.a = lora->a;
    a.b = lora->b;
    a.scale = lora->scale;
    a.adapter = adapter;
    a.row_start = row_start;
    a.n_adapters = lora->n_adapters;
    a.rank = lora->rank;
    a.k = lora->k;
    a.n = lora->n;
    a.n_req = n_req;
    a.max_tokens = rows;
    a.max_new = max_new;
    const long long tiles = tile_slots(rows, n_req, 1, 16);
    long long chunks = (1024 + tiles - 1) / tiles;
    const long long cap = ((long long)a.n + 127) / 128;
    if (chunks > cap) chunks = cap;
    if (chunks < 1) chunks = 1;
    a.chunk = (int)(((a.n + chunks - 1) / chunks + 127) / 128 * 128);
    const dim3 grid((unsigned)tiles, (unsigned)((a.n + a.chunk - 1) / a.chunk));
    hipStream_t st = stream_of(stream);
    if (x->dtype == NC_Q8) {
        if (out->dtype == NC_Q8) lora_launch<Q8, Q8>(a, grid, st);
        else if (out->dtype == NC_F16) lora_launch<Q8, F16>(a, grid, st);
        else lora_launch<Q8, F32>(a, grid, st);
    } else {
        if (out->dtype == NC_Q8) lora_launch<F16, Q8>(a, grid, st);
        else if (out->dtype == NC_F16) lora_launch<F16, F16>(a, grid, st);
        else lora_launch<F16, F32>(a, grid, st);
    }
    return launch_status("k_lora");
}
