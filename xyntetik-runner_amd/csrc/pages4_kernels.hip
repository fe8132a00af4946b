// Cache pages held in 4 bits (pages4.h has the format): rotating and writing a step's keys and values, reading rows and whole pages
// back, and attention over them for any head size in plain 32-bit arithmetic.
#include "pages4.h"

// ---------------------------------------------------------------- rotary + cache write
// Rotation as in k_rope_kv_write, of the angle pos * inv_freq itself: it is reduced to turns in 64 bits, so that far positions
// lose nothing (a 32-bit product is off by 0.004 at 131,071).
//
// A thread takes 8 channels of a head of queries, keys or values; 4 neighbouring lanes are a block of 32 and share its largest
// magnitude in two exchanges.  (A head's last block may be short: its missing lanes hold zeros.)  Where the rows are aligned it reads its channels and
// their partners in the rotation as four pieces of 16 bytes, before the angles are made.  A page holds the bytes of 8 positions of a value side by side: where the
// step brings such 8 positions whole, the workgroup of the first writes them all, 16 bytes at a time, and the other seven leave their values to it.
//
// Bound by memory: 2,048 tokens of 32 + 2 * 8 heads of 128 (50 MB of 32-bit rows in, 17 MB of queries and 2 MB of codes out) take 15.4 us, 4.5 TB/s where a
// large copy reaches 5.06 (channel by channel, a byte at a time and tokens in the order of their numbers 30.9); one token takes 2.8, the latency of its two
// dependent reads (position, page) and of the rows.
struct Write4Args {
    const float* q_in;      // [T, in_stride] 32-bit
    const float* k_in;
    const float* v_in;
    int in_stride;
    void* q_out;            // [T, H * D]
    Pages4 pages;
    const int* positions;   // [T]
    const int* req_of_token;
    const int* block_table; // [n_requests, table_width], rows table_stride apart
    int table_stride, table_width, n_requests, n_pages;
    const float* inv_freq;  // [rot / 2] or null
    int H, Hk, D, Dv, rot, interleaved, paired;
    float mscale;
    int page_shift, page_mask, page_size;
    int q_units, k_units, units, per_block;     // of a token: queries' end, keys' end, all; and those of a workgroup
    int lanes_k, lanes_v;                       // threads of a head of queries or keys, and of values (a multiple of 4, 32 at most)
    uint32_t per_k, per_v;                      // 2^32 over these, rounded up: a division below 2^26 is one product
    const float* bias;                          // SUMS: [columns of a row] or null
    size_t range_step;                          // SUMS: from a range's rows to the next's
    int ranges;
};

// (8 numbers of a row that begin at a multiple of 16 bytes)
template <typename T> __device__ inline void store_row8(T* dst, const float* v);
template <> __device__ inline void store_row8<float>(float* dst, const float* v) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <> __device__ inline void store_row8<bf16_t>(bf16_t* dst, const float* v) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

__device__ __forceinline__ void load_row8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// 8 sums of a product's K ranges, four ranges on their way at a time
__device__ __forceinline__ void load_sums8(const Write4Args& a, const float* p, const float* bias, float* v) {
    float b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b[i] = 0.f;
    if (bias) load_row8(bias, b);
    for (int s0 = 0; s0 < a.ranges; s0 += 4) {
        float part[4][8];
#pragma unroll
        for (int s = 0; s < 4; ++s) load_row8(p + (size_t)(s0 + s < a.ranges ? s0 + s : s0) * a.range_step, part[s]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += s0 + s < a.ranges ? part[s][i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
}
// the largest magnitude of a block of 32, of which the lane holds 8
__device__ __forceinline__ uint32_t most_of_block(const float* x) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1, 64));
    return max(most, (uint32_t)__shfl_xor((int)most, 2, 64));
}
// byte b of four words
template <int B> __device__ __forceinline__ uint32_t bytes_of(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
    const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x0c0c0400u + 0x0101u * B), hi = __builtin_amdgcn_perm(w3, w2, 0x04000c0cu + 0x01010000u * B);
    return lo | hi;
}

// VEC: rows of 16-byte pieces, and a rotation whose pairs lie in such pieces
// SUMS: a number is the sum of a product's K ranges, added in their order, and its column's bias: a kernel and a trip of the rows to memory less.  With the product,
// 32 + 2 * 8 heads of 128 behind 4,096 columns: 64 decoded tokens 20.3 us, in two kernels 21.3; 256 32.8 and 37.7; a prompt's 137 tokens 28.7 and 30.6.
template <typename T, bool VEC, bool SUMS>
__global__ __launch_bounds__(256) void k_rope_kv_write4(Write4Args a) {
    __shared__ float2 cs[8][17];                // pair j at [j % 8][j / 8]: lanes that read the i-th of their 8 pairs read side by side
    // (workgroups go to the eight dies in turn: 8 neighbouring tokens, whose codes share lines, to one of them)
    const int b = blockIdx.x, t = b < ((int)gridDim.x & ~63) ? (b & ~63) | (b & 7) << 3 | (b >> 3 & 7) : b;
    const int pos = a.positions[t];
    const int half = a.rot >> 1;
    const int u0 = blockIdx.y * a.per_block, u1 = min(a.units, u0 + a.per_block);
    const int req = a.req_of_token[t];
    // a unit: what it is, its head, its first channel, and its numbers as they come
    struct Unit { int h, c0, D; bool is_q, is_v; const float* src; float x[8], y[8]; };
    auto unit = [&](int u) __attribute__((always_inline)) {
        Unit w;
        w.is_q = u < a.q_units;
        w.is_v = u >= a.k_units;
        const int n = w.is_q ? u : w.is_v ? u - a.k_units : u - a.q_units, lanes = w.is_v ? a.lanes_v : a.lanes_k;
        w.D = w.is_v ? a.Dv : a.D;
        w.h = (int)__umulhi((unsigned)n, w.is_v ? a.per_v : a.per_k);         // n / lanes
        w.c0 = (n - w.h * lanes) * 8;
        w.src = (w.is_q ? a.q_in : w.is_v ? a.v_in : a.k_in) + (size_t)t * a.in_stride + (size_t)w.h * w.D;
        if constexpr (VEC) {
            const bool turn = !w.is_v && w.c0 < a.rot && !a.interleaved;
            int own = w.c0, other = w.c0;
            if (turn) {
                const bool second = w.c0 >= half;
                own = a.paired ? (second ? 2 * (w.c0 - half) + 8 : 2 * w.c0) : w.c0;
                other = a.paired ? (second ? own - 8 : own + 8) : second ? w.c0 - half : w.c0 + half;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) w.x[i] = w.y[i] = 0.f;
            if constexpr (SUMS) {
                const float* bias = a.bias ? a.bias + (w.src - a.q_in - (size_t)t * a.in_stride) : nullptr;
                if (w.c0 < w.D) load_sums8(a, w.src + own, bias ? bias + own : nullptr, w.x);
                if (turn) load_sums8(a, w.src + other, bias ? bias + other : nullptr, w.y);
            } else {
                if (w.c0 < w.D) load_row8(w.src + own, w.x);
                if (turn) load_row8(w.src + other, w.y);
            }
        }
        return w;
    };
    const int first = u0 + (int)threadIdx.x;
    Unit ahead = unit(first < u1 ? first : u0);
    for (int j = threadIdx.x; j < half; j += 256) {
        double turns = (double)pos * (double)a.inv_freq[j] * 0.15915494309189533577;
        turns -= rint(turns);
        // (what the angle loses as a 32-bit number is put back: cos(x + d) = cos x - d sin x, sin(x + d) = sin x + d cos x)
        const float x = (float)(2.0 * turns), d = (float)((2.0 * turns - x) * 3.14159265358979323846);
        float s, c;
        sincospif(x, &s, &c);
        cs[j & 7][j >> 3] = make_float2(fmaf(-d, s, c) * a.mscale, fmaf(d, c, s) * a.mscale);
    }
    const int bi = pos >> a.page_shift, off = pos & a.page_mask;
    const int page = bi >= 0 && bi < a.table_width && (unsigned)req < (unsigned)a.n_requests ? a.block_table[(size_t)req * a.table_stride + bi] : -1;
    const bool there = (unsigned)page < (unsigned)a.n_pages;          // (what has no page is written nowhere)
    // the 8 positions of a page that this one belongs to: whole in this step, row by row?
    const int lead = t - (pos & 7);
    bool whole = lead >= 0 && lead + 7 < (int)gridDim.x;
    if (whole)
#pragma unroll
        for (int i = 0; i < 8; ++i) whole &= a.req_of_token[lead + i] == req && a.positions[lead + i] == pos - (pos & 7) + i;
    __syncthreads();
    for (int u = first; u < u1; u += 256) {
        Unit w = u == first ? ahead : unit(u);
        float* x = w.x;
        if (w.is_v && whole) {
            if (pos & 7) continue;
            // 8 positions, all on their way at once: a word of codes each, then their bytes side by side
            uint32_t c[8], sc[2] = {0, 0};
            float v[8][8];
            const float* src = w.src + (w.c0 < w.D ? w.c0 : 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (VEC) load_row8(src + (size_t)i * a.in_stride, v[i]);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] = src[(size_t)i * a.in_stride + e];
            }
            if constexpr (SUMS) {
                for (int s = 1; s < a.ranges; ++s) {
                    float more[8][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) load_row8(src + (size_t)s * a.range_step + (size_t)i * a.in_stride, more[i]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[i][e] += more[i][e];
                }
                if (a.bias) {
                    float bias[8];
                    load_row8(a.bias + (src - a.q_in - (size_t)t * a.in_stride), bias);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[i][e] += bias[e];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (w.c0 >= w.D)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
                const uint32_t byte = scale_byte4(most_of_block(v[i]));
                c[i] = codes4(v[i], byte);
                sc[i >> 2] |= byte << (8 * (i & 3));
            }
            if (w.c0 >= w.D || !there) continue;
            const size_t pb = (size_t)page * a.Hk + w.h;
            if ((w.c0 & 31) == 0) *reinterpret_cast<uint2*>(a.pages.vs + scale_at4(pb, a.page_size, blocks4(w.D), off, w.c0 >> 5)) = make_uint2(sc[0], sc[1]);
            uint4* dst = reinterpret_cast<uint4*>(a.pages.vc + value_at4(pb, a.page_size, w.D, off, w.c0 >> 1));
            dst[0] = make_uint4(bytes_of<0>(c[0], c[1], c[2], c[3]), bytes_of<0>(c[4], c[5], c[6], c[7]), bytes_of<1>(c[0], c[1], c[2], c[3]), bytes_of<1>(c[4], c[5], c[6], c[7]));
            dst[1] = make_uint4(bytes_of<2>(c[0], c[1], c[2], c[3]), bytes_of<2>(c[4], c[5], c[6], c[7]), bytes_of<3>(c[0], c[1], c[2], c[3]), bytes_of<3>(c[4], c[5], c[6], c[7]));
            continue;
        }
        if constexpr (VEC) {
            if (!w.is_v && w.c0 < a.rot) {
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const int j = (w.c0 + i) >> 1;
                        const float2 r = cs[j & 7][j >> 3];
                        const float x0 = x[i], x1 = x[i + 1];
                        x[i] = x0 * r.x - x1 * r.y;
                        x[i + 1] = x0 * r.y + x1 * r.x;
                    }
                } else {
                    const bool second = w.c0 >= half;
                    const int j = second ? w.c0 - half : w.c0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 r = cs[i][j >> 3];
                        x[i] = second ? w.y[i] * r.y + x[i] * r.x : x[i] * r.x - w.y[i] * r.y;
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = w.c0 + i;
                if (w.c0 >= w.D) {
                    x[i] = 0.f;
                } else if (w.is_v || c >= a.rot) {
                    x[i] = w.src[c];
                } else {
                    const int j = a.interleaved ? c >> 1 : c < half ? c : c - half;
                    const bool second = a.interleaved ? (c & 1) : c >= half;
                    int i0 = a.interleaved ? 2 * j : j, i1 = a.interleaved ? 2 * j + 1 : j + half;
                    if (a.paired) { i0 = paired_col(i0, a.rot); i1 = paired_col(i1, a.rot); }
                    const float x0 = w.src[i0], x1 = w.src[i1];
                    const float2 r = cs[j & 7][j >> 3];
                    x[i] = second ? x0 * r.y + x1 * r.x : x0 * r.x - x1 * r.y;
                }
            }
        }
        if (w.is_q) {
            if (w.c0 < w.D) store_row8<T>((T*)a.q_out + ((size_t)t * a.H + w.h) * w.D + w.c0, x);
            continue;
        }
        const uint32_t most = most_of_block(x);
        if (w.c0 >= w.D || !there) continue;
        const uint32_t byte = scale_byte4(most), codes = codes4(x, byte);
        const size_t pb = (size_t)page * a.Hk + w.h;
        uint8_t* scales = w.is_v ? a.pages.vs : a.pages.ks;
        if ((w.c0 & 31) == 0) scales[scale_at4(pb, a.page_size, blocks4(w.D), off, w.c0 >> 5)] = (uint8_t)byte;
        if (w.is_v) {
            uint8_t* dst = a.pages.vc + value_at4(pb, a.page_size, w.D, off, w.c0 >> 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[8 * i] = (uint8_t)(codes >> (8 * i));
        } else {
            *reinterpret_cast<uint32_t*>(a.pages.kc + key_at4(pb, a.page_size, w.D, off) + (w.c0 >> 1)) = codes;
        }
    }
}

static int check_pages4(const char* what, const Pages4& p, int Hk, int D, int Dv, int page_size, int n_pages) {
    XR_REQUIRE(Hk > 0 && D > 0 && Dv > 0 && D <= 256 && Dv <= 256 && D % 8 == 0 && Dv % 8 == 0,
               "%s: 4-bit pages hold heads of 8 to 256 channels in steps of 8, not %d keys and values of %d and %d", what, Hk, D, Dv);
    XR_REQUIRE(ilog2_exact(page_size) >= 3, "%s: 4-bit pages have a power of two of at least 8 positions, not %d", what, page_size);
    XR_REQUIRE(p.kc && p.ks && p.vc && p.vs && n_pages > 0, "%s: 4-bit pages with a null operand", what);
    XR_REQUIRE((((uintptr_t)p.kc | (uintptr_t)p.vc) & 15) == 0 && (((uintptr_t)p.ks | (uintptr_t)p.vs) & 7) == 0,
               "%s: 4-bit pages must be 16-byte aligned, their scales 8-byte", what);
    return XR_OK;
}

// the work of a token in workgroups: one where there are tokens enough for the chip, else a round of threads each
static dim3 deal_units(Write4Args& a, int T) {
    a.lanes_k = blocks4(a.D) * 4; a.lanes_v = blocks4(a.Dv) * 4;
    a.per_k = (uint32_t)(((1ull << 32) + a.lanes_k - 1) / a.lanes_k); a.per_v = (uint32_t)(((1ull << 32) + a.lanes_v - 1) / a.lanes_v);
    a.q_units = a.H * a.lanes_k; a.k_units = a.q_units + a.Hk * a.lanes_k; a.units = a.k_units + a.Hk * a.lanes_v;
    int groups = (1024 + T - 1) / T;
    const int most = (a.units + 255) / 256;
    groups = groups < 1 ? 1 : groups > most ? most : groups;
    a.per_block = ((a.units + groups - 1) / groups + 255) / 256 * 256;
    return dim3(T, (a.units + a.per_block - 1) / a.per_block);
}

int rope_kv_write4_sums(const Write4Sums& w, hipStream_t stream) {
    const XrGemmPages4& p = *w.pages;
    Write4Args a;
    a.pages = Pages4{(uint8_t*)p.kc, (uint8_t*)p.ks, (uint8_t*)p.vc, (uint8_t*)p.vs};
    const int rc = check_pages4("gemm", a.pages, w.Hk, w.D, w.D, w.page_size, p.n_pages);
    if (rc != XR_OK) return rc;
    a.in_stride = (w.H + 2 * w.Hk) * w.D;
    XR_REQUIRE(a.in_stride % 4 == 0 && (((uintptr_t)w.sums | (uintptr_t)w.bias | (uintptr_t)w.q_out) & 15) == 0 && (w.interleaved ? w.rot % 8 == 0 : w.rot % 16 == 0),
               "gemm: rows that go to 4-bit pages must be 16-byte aligned, their rotary width (%d) a multiple of 16 (pairs of neighbours: 8)", w.rot);
    a.q_in = w.sums; a.k_in = w.sums + (size_t)w.H * w.D; a.v_in = a.k_in + (size_t)w.Hk * w.D; a.q_out = w.q_out;
    a.bias = w.bias; a.range_step = (size_t)w.T * a.in_stride; a.ranges = w.ranges;
    a.positions = w.positions; a.req_of_token = w.req_of_token; a.block_table = w.block_table; a.table_stride = w.table_stride;
    a.table_width = p.table_width; a.n_requests = p.n_requests; a.n_pages = p.n_pages; a.inv_freq = w.inv_freq; a.H = w.H; a.Hk = w.Hk; a.D = a.Dv = w.D; a.rot = w.rot;
    a.interleaved = w.interleaved; a.paired = !w.interleaved && w.rot > 0; a.mscale = w.mscale;
    a.page_shift = ilog2_exact(w.page_size); a.page_mask = w.page_size - 1; a.page_size = w.page_size;
    const dim3 grid = deal_units(a, w.T);
    k_rope_kv_write4<bf16_t, true, true><<<grid, 256, 0, stream>>>(a);
    XR_CHECK_LAUNCH("rope_kv_write4_sums");
    return XR_OK;
}

extern "C" int xr_rope_kv_write4(const float* q_in, const float* k_in, const float* v_in, int in_stride, void* q_out,
                                 void* kc, void* ks, void* vc, void* vs, int n_pages, const int* positions, const int* req_of_token,
                                 const int* block_table, int table_stride, int table_width, int n_requests, const float* inv_freq, int T, int H, int Hk,
                                 int D, int Dv, int rot, int interleaved, float mscale, int page_size, int q_dtype, int paired,
                                 hipStream_t stream) {
    Write4Args a;
    a.pages = Pages4{(uint8_t*)kc, (uint8_t*)ks, (uint8_t*)vc, (uint8_t*)vs};
    const int rc = check_pages4("rope_kv_write", a.pages, Hk, D, Dv, page_size, n_pages);
    if (rc != XR_OK) return rc;
    XR_REQUIRE(T >= 0 && H >= 0 && H < (1 << 20) && Hk < (1 << 20) && table_stride >= 0 && table_width > 0, "rope_kv_write: bad sizes T=%d H=%d, block tables of %d pages", T, H, table_width);
    XR_REQUIRE(rot >= 0 && rot <= D && rot % 2 == 0, "rope_kv_write: rotary width %d must be even and at most head_dim %d", rot, D);
    XR_REQUIRE(rot == 0 || inv_freq, "rope_kv_write: rotary width %d without a frequency table", rot);
    XR_REQUIRE(q_dtype == XR_F32 || q_dtype == XR_BF16, "rope_kv_write: bad dtype %d", q_dtype);
    XR_REQUIRE(!paired || (!interleaved && rot % 16 == 0), "rope_kv_write: paired order needs pairs (j, j + width/2) and a rotary width (%d) that is a multiple of 16", rot);
    if (T == 0) return XR_OK;
    XR_REQUIRE(k_in && v_in && block_table && req_of_token && positions, "rope_kv_write: keys and values to cache but a null operand");
    XR_REQUIRE(H == 0 || (q_in && q_out && ((uintptr_t)q_out & 15) == 0), "rope_kv_write: queries but a null operand, or rows that are not 16-byte aligned");
    a.q_in = q_in; a.k_in = k_in; a.v_in = v_in; a.in_stride = in_stride; a.q_out = q_out; a.bias = nullptr; a.range_step = 0; a.ranges = 1;
    a.positions = positions; a.req_of_token = req_of_token; a.block_table = block_table; a.table_stride = table_stride; a.table_width = table_width; a.n_requests = n_requests; a.n_pages = n_pages;
    a.inv_freq = inv_freq; a.H = H; a.Hk = Hk; a.D = D; a.Dv = Dv; a.rot = rot; a.interleaved = interleaved; a.paired = paired ? 1 : 0;
    a.mscale = mscale; a.page_shift = ilog2_exact(page_size); a.page_mask = page_size - 1; a.page_size = page_size;
    const dim3 grid = deal_units(a, T);
    const bool vec = in_stride % 4 == 0 && (((uintptr_t)(H ? q_in : k_in) | (uintptr_t)k_in | (uintptr_t)v_in) & 15) == 0 && (interleaved ? rot % 8 == 0 : rot % 16 == 0);
    if (q_dtype == XR_F32) {
        if (vec) k_rope_kv_write4<float, true, false><<<grid, 256, 0, stream>>>(a);
        else k_rope_kv_write4<float, false, false><<<grid, 256, 0, stream>>>(a);
    } else if (vec) k_rope_kv_write4<bf16_t, true, false><<<grid, 256, 0, stream>>>(a);
    else k_rope_kv_write4<bf16_t, false, false><<<grid, 256, 0, stream>>>(a);
    XR_CHECK_LAUNCH("rope_kv_write4");
    return XR_OK;
}

// ---------------------------------------------------------------- reading back
// 8 channels of one position, the lowest of them c0 (a multiple of 8)
__device__ inline void key_row8(const Pages4& p, size_t pb, int page_size, int D, int off, int c0, float* x) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p.kc + key_at4(pb, page_size, D, off) + (c0 >> 1));
    const uint32_t s = (uint32_t)p.ks[scale_at4(pb, page_size, blocks4(D), off, c0 >> 5)] << 23;
    const float2 v[4] = {pair4_f32<0>(w, s), pair4_f32<1>(w, s), pair4_f32<2>(w, s), pair4_f32<3>(w, s)};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = v[i].x; x[2 * i + 1] = v[i].y; }
}
__device__ inline void value_row8(const Pages4& p, size_t pb, int page_size, int Dv, int off, int c0, float* x) {
    const uint32_t s = (uint32_t)p.vs[scale_at4(pb, page_size, blocks4(Dv), off, c0 >> 5)] << 23;
    const uint8_t* src = p.vc + value_at4(pb, page_size, Dv, off, c0 >> 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = pair4_f32<0>((uint32_t)src[8 * i], s);
        x[2 * i] = v.x; x[2 * i + 1] = v.y;
    }
}

struct Read4Args {
    Pages4 pages;
    const int* positions;       // rows: [n]
    const int* req_of_row;
    const int* block_table;
    const int* slots;           // pages: [n, 3] request, place in its table, positions of the page that are the request's
    void* k_out;                // rows: [n, Hk * D]; pages: [n, Hk, page_size, D]
    void* v_out;                // rows: [n, Hk * Dv]; pages: [n, Hk, Dv, page_size]
    int table_stride, table_width, n_requests, n_pages, Hk, D, Dv, page_shift, page_size;
    size_t total;               // threads of all rows, keys' first
    size_t k_total;
};

// Rows of a list of (request, position): a thread 8 channels of a head, whose codes are one word (of a value: 4 bytes 8 apart, in lines that the row's neighbours
// share).  Rows without a page read as zeros.  2,048 rows of 8 heads of 128, 16 bits, take 7.2 us for 9.5 MB, 1.3 TB/s of the 5.06 of a large copy: not memory, but three trips that wait for one
// another (position, page, codes: one row takes 2.5) and a value's codes byte by byte.
template <typename T>
__global__ __launch_bounds__(256) void k_read_rows4(Read4Args a) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < a.total; i += (size_t)gridDim.x * 256) {
        const bool is_v = i >= a.k_total;
        const int D = is_v ? a.Dv : a.D, per = a.Hk * (D >> 3);
        const size_t j = is_v ? i - a.k_total : i;
        const size_t r = j / per;
        const int w = (int)(j - r * per), h = w / (D >> 3), c0 = (w - h * (D >> 3)) * 8;
        const int pos = a.positions[r], bi = pos >> a.page_shift, off = pos & (a.page_size - 1);
        const int req = a.req_of_row[r];
        const int page = bi >= 0 && bi < a.table_width && (unsigned)req < (unsigned)a.n_requests ? a.block_table[(size_t)req * a.table_stride + bi] : -1;
        float x[8];
        if ((unsigned)page >= (unsigned)a.n_pages) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
        } else {
            const size_t pb = (size_t)page * a.Hk + h;
            if (is_v) value_row8(a.pages, pb, a.page_size, D, off, c0, x);
            else key_row8(a.pages, pb, a.page_size, D, off, c0, x);
        }
        store_row8<T>((T*)(is_v ? a.v_out : a.k_out) + (r * a.Hk + h) * D + c0, x);
    }
}

// Whole pages in the layout of 16- and 32-bit caches (values transposed), a workgroup a page and head.  What lies behind a request's
// end becomes zero, so that readers may multiply it.  Bound by memory: 32,768 positions of 8 heads of 128 (36 MB in, 134 MB out, 16 bits) take 37 us, 4.6 TB/s, and 27.4 where the results of a call before lie in the last cache;
// 13,300 of 8 heads of 64 in 32 bits (7 MB in, 55 MB out) 13.5, 4.6 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void k_read_pages4(Read4Args a) {
    const int n = blockIdx.x / a.Hk, h = blockIdx.x - n * a.Hk;
    const int req = a.slots[3 * n], bi = a.slots[3 * n + 1], held = a.slots[3 * n + 2];
    const int page = a.block_table[(size_t)req * a.table_stride + bi];
    const bool there = (unsigned)page < (unsigned)a.n_pages;
    const size_t pb = (size_t)(there ? page : 0) * a.Hk + h, to = (size_t)n * a.Hk + h;
    const int P = a.page_size, oct = a.D >> 3;
    for (int i = threadIdx.x; i < P * oct; i += 256) {
        const int off = i / oct, c0 = (i - off * oct) * 8;
        float x[8];
        key_row8(a.pages, pb, P, a.D, off, c0, x);
        if (!there || off >= held)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
        store_row8<T>((T*)a.k_out + (to * P + off) * a.D + c0, x);
    }
    // values: a thread 8 positions of two channels
    const int octs = P >> 3;
    for (int i = threadIdx.x; i < octs * (a.Dv >> 1); i += 256) {
        const int pair = i / octs, o8 = i - pair * octs;
        const uint2 w = *reinterpret_cast<const uint2*>(a.pages.vc + value_at4(pb, P, a.Dv, o8 * 8, pair));
        const uint2 s = *reinterpret_cast<const uint2*>(a.pages.vs + scale_at4(pb, P, blocks4(a.Dv), o8 * 8, pair >> 4));
        const float2 v[8] = {pair4_f32<0>(w.x, s.x << 23), pair4_f32<1>(w.x, s.x << 15), pair4_f32<2>(w.x, s.x << 7), pair4_f32<3>(w.x, s.x >> 1),
                             pair4_f32<0>(w.y, s.y << 23), pair4_f32<1>(w.y, s.y << 15), pair4_f32<2>(w.y, s.y << 7), pair4_f32<3>(w.y, s.y >> 1)};
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool ok = there && o8 * 8 + e < held;
            x[e] = ok ? v[e].x : 0.f;
            y[e] = ok ? v[e].y : 0.f;
        }
        T* dst = (T*)a.v_out + (to * a.Dv + 2 * pair) * P + o8 * 8;
        store_row8<T>(dst, x);
        store_row8<T>(dst + P, y);
    }
}

extern "C" int xr_read_rows4(void* k_out, void* v_out, void* kc, void* ks, void* vc, void* vs, int n_pages, const int* positions,
                             const int* req_of_row, const int* block_table, int table_stride, int table_width, int n_requests, int n, int Hk, int D,
                             int Dv, int page_size, int dtype, hipStream_t stream) {
    Read4Args a;
    a.pages = Pages4{(uint8_t*)kc, (uint8_t*)ks, (uint8_t*)vc, (uint8_t*)vs};
    const int rc = check_pages4("read_rows", a.pages, Hk, D, Dv, page_size, n_pages);
    if (rc != XR_OK) return rc;
    XR_REQUIRE(n >= 0 && table_stride >= 0 && table_width > 0 && (dtype == XR_F32 || dtype == XR_BF16), "read_rows: bad sizes n=%d table=%d or dtype %d", n, table_width, dtype);
    if (n == 0) return XR_OK;
    XR_REQUIRE(k_out && v_out && positions && req_of_row && block_table, "read_rows: a null operand");
    XR_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "read_rows: outputs must be 16-byte aligned");
    a.positions = positions; a.req_of_row = req_of_row; a.block_table = block_table; a.slots = nullptr;
    a.k_out = k_out; a.v_out = v_out; a.table_stride = table_stride; a.table_width = table_width; a.n_requests = n_requests; a.n_pages = n_pages; a.Hk = Hk; a.D = D; a.Dv = Dv;
    a.page_shift = ilog2_exact(page_size); a.page_size = page_size;
    a.k_total = (size_t)n * Hk * (D >> 3);
    a.total = a.k_total + (size_t)n * Hk * (Dv >> 3);
    const size_t blocks = (a.total + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
    if (dtype == XR_F32) k_read_rows4<float><<<grid, 256, 0, stream>>>(a);
    else k_read_rows4<bf16_t><<<grid, 256, 0, stream>>>(a);
    XR_CHECK_LAUNCH("read_rows4");
    return XR_OK;
}

extern "C" int xr_read_pages4(void* k_out, void* v_out, void* kc, void* ks, void* vc, void* vs, int n_pages, const int* slots, int n,
                              const int* block_table, int table_stride, int Hk, int D, int Dv, int page_size, int dtype, hipStream_t stream) {
    Read4Args a;
    a.pages = Pages4{(uint8_t*)kc, (uint8_t*)ks, (uint8_t*)vc, (uint8_t*)vs};
    const int rc = check_pages4("read_pages", a.pages, Hk, D, Dv, page_size, n_pages);
    if (rc != XR_OK) return rc;
    XR_REQUIRE(n >= 0 && table_stride > 0 && (dtype == XR_F32 || dtype == XR_BF16), "read_pages: bad sizes n=%d table=%d or dtype %d", n, table_stride, dtype);
    if (n == 0) return XR_OK;
    XR_REQUIRE((long long)n * Hk < (1LL << 31), "read_pages: %d pages of %d heads are more workgroups than a launch takes", n, Hk);
    XR_REQUIRE(k_out && v_out && slots && block_table, "read_pages: a null operand");
    XR_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "read_pages: outputs must be 16-byte aligned");
    a.positions = nullptr; a.req_of_row = nullptr; a.block_table = block_table; a.slots = slots;
    a.k_out = k_out; a.v_out = v_out; a.table_stride = table_stride; a.table_width = a.n_requests = 0; a.n_pages = n_pages; a.Hk = Hk; a.D = D; a.Dv = Dv;
    a.page_shift = ilog2_exact(page_size); a.page_size = page_size; a.total = a.k_total = 0;
    const unsigned grid = (unsigned)n * (unsigned)Hk;
    if (dtype == XR_F32) k_read_pages4<float><<<grid, 256, 0, stream>>>(a);
    else k_read_pages4<bf16_t><<<grid, 256, 0, stream>>>(a);
    XR_CHECK_LAUNCH("read_pages4");
    return XR_OK;
}

// ---------------------------------------------------------------- attention, any head size
// Attention over 4-bit pages in 32 bits: a workgroup a token and query head, its waves 64 keys a turn each; a key a lane for the scores, a pair of channels a
// lane for the values, 8 positions at a time as they lie side by side; the options of k_attention_ref.  For what the matrix-core kernel does not take: 32-bit
// queries of few rows, head sizes that end inside a block and, in recorded steps, whose pages cannot be read back first, the other sizes and kept first keys.
//
// Bound by instructions as the work is shared out: every query head converts its keys and values again (and a request's keys are not cut into ranges: few requests leave compute units idle), and beside a product stand half a conversion and the shared memory's reads of the
// query.  8 requests of 4,000 keys, 32 heads of 128 over 8, take 57 us (9 TFLOP/s; channel by channel with a byte a load 252), 64 of 8,000 with heads of 64 344 (12 TFLOP/s).
#define ANY4_WAVES 8
struct Any4Args {
    Pages4 pages;
    const void* q;              // [T, H * D]
    void* out;                  // [T, H, Dv], rows ld_out apart
    const int* positions;
    const int* req_of_token;
    const int* block_table;
    const float* slopes;
    const float* sinks;
    const float* gate;
    int table_stride, n_pages, H, Hk, D, Dv, page_shift, page_size, window, chunk, keep, ld_gate, ld_out;
    float scale, cap, out_scale;
};

// WIDE: keys in whole blocks, a block's codes in one load
template <typename T, bool WIDE>
__global__ __launch_bounds__(64 * ANY4_WAVES) void k_attention_any4(Any4Args a) {
    __shared__ __align__(16) float qs[256];
    __shared__ float sums[ANY4_WAVES][256], ml[ANY4_WAVES][2];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pos = a.positions[t], kvh = h / (a.H / a.Hk);
    const int lo = a.chunk > 0 ? pos - pos % a.chunk : (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
    const int kept = a.keep < lo ? a.keep : lo;
    for (int d = threadIdx.x; d < a.D; d += 64 * ANY4_WAVES) qs[d] = ld<T>((const T*)a.q, ((size_t)t * a.H + h) * a.D + d);
    __syncthreads();
    const int* bt = a.block_table + (size_t)a.req_of_token[t] * a.table_stride;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    const int P = a.page_size, nbk = blocks4(a.D), nbv = blocks4(a.Dv), pairs = a.Dv >> 1;
    const bool both = pairs <= 32;                  // few pairs: the halves of a wave take turns with the eights of positions
    const int pair = both ? lane & 31 : lane;
    float m = -INFINITY, l = 0.f;
    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    for (int seg = kept > 0 ? 0 : 1; seg < 2; ++seg) {
        const int begin = seg ? lo : 0, last = seg ? pos : kept - 1;
        for (int k0 = (begin & ~7) + 64 * wave; k0 <= last; k0 += 64 * ANY4_WAVES) {
            const int key = k0 + lane, bi = key >> a.page_shift;
            int page = key <= last && bi < a.table_stride ? bt[bi] : -1;       // (a place past the table, or a page that was given back: none)
            page = (unsigned)page < (unsigned)a.n_pages ? page : -1;
            const bool seen = page >= 0 && key >= begin;
            float s = -INFINITY;
            if (seen) {
                const size_t pb = (size_t)page * a.Hk + kvh;
                const int off = key & (P - 1);
                const uint8_t* codes = a.pages.kc + key_at4(pb, P, a.D, off);
                const uint8_t* scales = a.pages.ks + scale_at4(pb, P, nbk, off, 0);
                float dot = 0.f;
                for (int b = 0; b < nbk; ++b) {
                    const uint32_t sc = (uint32_t)scales[8 * b] << 23;
                    uint32_t w[4];
                    const int n = WIDE ? 4 : min(4, (a.D - 32 * b) >> 3);
                    if constexpr (WIDE) {
                        const uint4 v = *reinterpret_cast<const uint4*>(codes + 16 * b);
                        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = i < n ? *reinterpret_cast<const uint32_t*>(codes + 16 * b + 4 * i) : 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!WIDE && i >= n) break;
                        const float4 qa = *reinterpret_cast<const float4*>(qs + 32 * b + 8 * i), qb = *reinterpret_cast<const float4*>(qs + 32 * b + 8 * i + 4);
                        const float2 v0 = pair4_f32<0>(w[i], sc), v1 = pair4_f32<1>(w[i], sc), v2 = pair4_f32<2>(w[i], sc), v3 = pair4_f32<3>(w[i], sc);
                        dot = fmaf(qa.x, v0.x, dot); dot = fmaf(qa.y, v0.y, dot); dot = fmaf(qa.z, v1.x, dot); dot = fmaf(qa.w, v1.y, dot);
                        dot = fmaf(qb.x, v2.x, dot); dot = fmaf(qb.y, v2.y, dot); dot = fmaf(qb.z, v3.x, dot); dot = fmaf(qb.w, v3.y, dot);
                    }
                }
                s = dot * a.scale;
                if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
                s -= slope * (float)(pos - key);
            }
            const float mn = fmaxf(m, wave_max(s));
            const float p = seen ? expf(s - mn) : 0.f;
            const float corr = m == -INFINITY ? 0.f : expf(m - mn);
            l = l * corr + wave_sum(p);
            m = mn;
#pragma unroll
            for (int i = 0; i < 2; ++i) { acc[i].x *= corr; acc[i].y *= corr; }
            const unsigned long long mask = __ballot(seen);
            if (!mask) continue;
            for (int o = 0; o < 8; o += both ? 2 : 1) {
                const int mine = both ? o + (lane >> 5) : o;
                const uint32_t some = (uint32_t)(mask >> (8 * mine)) & 255u;
                const int pg = __shfl(page, 8 * mine + (some ? __ffs((int)some) - 1 : 0), 64);
                float pj[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) pj[e] = __shfl(p, 8 * mine + e, 64);
                if (!some) continue;
                const size_t pb = (size_t)pg * a.Hk + kvh;
                const int off = (k0 + 8 * mine) & (P - 1);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int pr = pair + 64 * i;
                    if (pr >= pairs || (i > 0 && both)) break;
                    const uint2 c = *reinterpret_cast<const uint2*>(a.pages.vc + value_at4(pb, P, a.Dv, off, pr));
                    const uint2 sc = *reinterpret_cast<const uint2*>(a.pages.vs + scale_at4(pb, P, nbv, off, pr >> 4));
                    // (a position that is not seen is no number's: its scale becomes the smallest, its weight is 0)
                    const float2 v[8] = {pair4_f32<0>(c.x, some & 1 ? sc.x << 23 : 0u), pair4_f32<1>(c.x, some & 2 ? sc.x << 15 : 0u),
                                         pair4_f32<2>(c.x, some & 4 ? sc.x << 7 : 0u), pair4_f32<3>(c.x, some & 8 ? sc.x >> 1 : 0u),
                                         pair4_f32<0>(c.y, some & 16 ? sc.y << 23 : 0u), pair4_f32<1>(c.y, some & 32 ? sc.y << 15 : 0u),
                                         pair4_f32<2>(c.y, some & 64 ? sc.y << 7 : 0u), pair4_f32<3>(c.y, some & 128 ? sc.y >> 1 : 0u)};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        acc[i].x = fmaf(pj[e], v[e].x, acc[i].x);
                        acc[i].y = fmaf(pj[e], v[e].y, acc[i].y);
                    }
                }
            }
        }
    }
    if (both) {
        acc[0].x += __shfl_xor(acc[0].x, 32, 64);
        acc[0].y += __shfl_xor(acc[0].y, 32, 64);
    }
    // the waves' shares in one scale (a wave without keys has the sum 0)
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (pair + 64 * i < pairs && !(both && (i > 0 || lane > 31))) {
            sums[wave][2 * (pair + 64 * i)] = acc[i].x;
            sums[wave][2 * (pair + 64 * i) + 1] = acc[i].y;
        }
    if (lane == 0) {
        ml[wave][0] = m;
        ml[wave][1] = l;
    }
    __syncthreads();
    float most = a.sinks ? a.sinks[h] : -INFINITY;
    for (int w = 0; w < ANY4_WAVES; ++w) most = fmaxf(most, ml[w][0]);
    float all = a.sinks ? expf(a.sinks[h] - most) : 0.f;
    for (int w = 0; w < ANY4_WAVES; ++w) all += ml[w][1] == 0.f ? 0.f : ml[w][1] * expf(ml[w][0] - most);
    const float f = a.gate ? a.out_scale / (1.0f + expf(-a.gate[(size_t)t * a.ld_gate + h])) : a.out_scale;
    T* orow = (T*)a.out + (size_t)t * a.ld_out + (size_t)h * a.Dv;
    for (int d = threadIdx.x; d < a.Dv; d += 64 * ANY4_WAVES) {
        float o = 0.f;
        for (int w = 0; w < ANY4_WAVES; ++w) o += ml[w][1] == 0.f ? 0.f : sums[w][d] * expf(ml[w][0] - most);
        st<T>(orow, d, all == 0.f ? 0.f : o / all * f);      // (0: no key that exists and no sink)
    }
}

extern "C" int xr_attention_any4(void* out, const void* q, void* kc, void* ks, void* vc, void* vs, int n_pages, const int* positions,
                                 const int* req_of_token, const int* block_table, int table_stride, int T, int H, int Hk, int D, int Dv,
                                 int page_size, float scale, int window, int chunk, int keep, int dtype, const float* slopes,
                                 const float* sinks, float cap, const float* gate, int ld_gate, float out_scale, int ld_out,
                                 hipStream_t stream) {
    Any4Args a;
    a.pages = Pages4{(uint8_t*)kc, (uint8_t*)ks, (uint8_t*)vc, (uint8_t*)vs};
    const int rc = check_pages4("attention", a.pages, Hk, D, Dv, page_size, n_pages);
    if (rc != XR_OK) return rc;
    XR_REQUIRE(T >= 0 && H > 0 && H <= 65535 && H % Hk == 0, "attention: %d query heads are not a multiple of %d key/value heads (65,535 at most)", H, Hk);
    XR_REQUIRE(window >= 0 && chunk >= 0 && keep >= 0 && !(window && chunk), "attention: window %d, chunk %d or kept keys %d", window, chunk, keep);
    XR_REQUIRE(cap >= 0.f, "attention: soft cap %g is negative", (double)cap);
    XR_REQUIRE(ld_out >= H * Dv && (!gate || ld_gate >= H), "attention: output rows %d apart, a gate's %d", ld_out, ld_gate);
    XR_REQUIRE(dtype == XR_F32 || dtype == XR_BF16, "attention: bad dtype %d", dtype);
    if (T == 0) return XR_OK;
    XR_REQUIRE(out && q && positions && req_of_token && block_table && table_stride > 0, "attention: a null operand");
    a.q = q; a.out = out; a.positions = positions; a.req_of_token = req_of_token; a.block_table = block_table;
    a.slopes = slopes; a.sinks = sinks; a.gate = gate; a.table_stride = table_stride; a.n_pages = n_pages; a.H = H; a.Hk = Hk;
    a.D = D; a.Dv = Dv; a.page_shift = ilog2_exact(page_size); a.page_size = page_size; a.window = window; a.chunk = chunk; a.keep = keep;
    a.ld_gate = ld_gate; a.ld_out = ld_out; a.scale = scale; a.cap = cap; a.out_scale = out_scale;
    const dim3 grid(T, H);
    if (dtype == XR_F32) {
        if (D % 32 == 0) k_attention_any4<float, true><<<grid, 64 * ANY4_WAVES, 0, stream>>>(a);
        else k_attention_any4<float, false><<<grid, 64 * ANY4_WAVES, 0, stream>>>(a);
    } else if (D % 32 == 0) k_attention_any4<bf16_t, true><<<grid, 64 * ANY4_WAVES, 0, stream>>>(a);
    else k_attention_any4<bf16_t, false><<<grid, 64 * ANY4_WAVES, 0, stream>>>(a);
    XR_CHECK_LAUNCH("attention_any4");
    return XR_OK;
}
