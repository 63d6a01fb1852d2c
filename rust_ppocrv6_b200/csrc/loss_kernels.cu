// sm_100a kernels of the recognition head's training losses: softmax cross entropy over the CTC
// vocabulary and distillation from a teacher's top logits, without the [rows][classes] logits in
// memory. Both hold the row's softmax p = softmax(z / T), z = x W^T + b, against a sparse
// distribution q (one class, or the teacher's entries), so they share every kernel:
//
//   loss_r = T^2 sum_i q_i (log q_i - log p[c_i]),   dz_r = T g_r (p - q),
//   dx = dz W,  dW = dz^T x,  db = sum_r dz_r        (cross entropy: q = 1 at the target, T = 1)
//
//  loss_pack_kernel    operand tiles of 128 rows as tensor-core images, labels sorted by class tile
//  loss_main_kernel    the dense work, in one of two directions that mirror each other:
//                        row pass    own = 128 rows of x, streamed = W tiles: running (max, sum) of
//                                    the softmax and sum_j p_j W_j, over the classes that the row
//                                    does not name
//                        weight pass own = 128 classes, streamed = x tiles: dz^T x with p from the
//                                    rows' lse, and dz of the named classes as the row kernel left it
//  loss_rows_kernel    joins a row's class ranges and adds the named classes: loss, lse, their dz, dx
//  loss_reduce_kernel  joins a class's row ranges: dW, db
//  loss_score_kernel   loss and lse of a packed head from the decode kernel's (argmax, probability)
//
// The classes that a row names are kept out of the dense products, because there p - q cancels: a row
// whose target has p = 0.9999 has a gradient of 1e-4 of p, and p rounded to bf16 (2^-9), or added up by
// a tensor core that rounds toward zero (2^-23 a step), would be off by more than that. The row kernel
// forms their logits in f32 and takes 1 - p as what it is, the other classes' share. (With the named
// classes in the products, da of rows with p of 0.9 to 0.99999 was 10 to 50,000 times further off.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "head_params.h"
#include "loss_params.h"
#include "loss_ptx.cuh"

namespace rh {

namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <bool F32>
struct Elem {
    using type = float;
};
template <>
struct Elem<false> {
    using type = __nv_bfloat16;
};

// Byte offset of 16-byte chunk `ch` (8 K slots) of row r in a 128 x 128 16-bit tile image: two
// halves of 64 K slots, rows of 128 bytes, chunks XOR-swizzled by the row (the tensor core's
// 128-byte swizzle).
__device__ __forceinline__ uint32_t image_chunk(int r, int ch) {
    return (uint32_t)(ch >> 3) * 16384u + (uint32_t)r * 128u + (uint32_t)(((ch & 7) ^ (r & 7)) << 4);
}

// Where element (row, kk) of the features lies: rows of k, or the SVTR tail's [b][k][t_len].
__device__ __forceinline__ long long x_base(long long row, int k, long long t_len) {
    return t_len > 0 ? (row / t_len) * (long long)k * t_len + row % t_len : row * (long long)k;
}

// Exponent of the power of two that brings `top` (> 0, finite) into [2^target, 2^(target + 1)).
__device__ __forceinline__ int shift_to(float top, int target) {
    if (!(top > 0.0f) || top > 3.4028235e38f) return 0;
    const int e = (int)((__float_as_uint(top) >> 23) & 0xFFu) - 127;
    return min(max(target - e, -126), 126);
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// What an earlier kernel of the same chain wrote. The kernel that reads it may have been resident since
// before the write (launch_next), so it is no read-only data: the non-coherent path of __ldg could return
// a line that this SM's L1 kept of the same address, as one workspace part serves one kernel after the
// other. Read from L2. (__ldg is for what the caller brings: weight, bias, packed tiles.)
template <class T>
__device__ __forceinline__ T chain_load(const T* p) {
    return __ldcg(p);
}
__device__ __forceinline__ float2 as_pair(uint32_t a, uint32_t b) {
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
// Whether class c is one of a row's labels at all.
__device__ __forceinline__ bool is_class(int c, int n) { return c >= 0 && c < n; }

}  // namespace

// ------------------------------------------------------------------------------------ pack
// One block per tile: w_tiles weight tiles, then x_tiles feature tiles. f32 values are scaled by
// the tile's power of two into [2^14, 2^15) and split into fp16 hi + lo (~22 bits below the
// tile's maximum, which an image of fp16 alone or of bf16 parts would not hold); bf16 values are
// copied. A row that is ignored is zero in the image, so whatever its features hold (NaN
// included) reaches nothing.
// The labels of a feature tile are sorted by 32 classes (a softmax warp's), rows ascending: each
// warp takes 8 rows, a group of lanes per row, and notes for every entry how many of its bin came
// before it in the warp; a scan over warps and bins then gives every entry its place (no atomics:
// the order is fixed). A class that a row names twice has one place, its first entry's.
constexpr int kPackThreads = 512, kPackWarps = kPackThreads / 32, kPackItems = 2048 / kPackThreads;

template <bool F32>
__global__ void __launch_bounds__(kPackThreads, 2) loss_pack_kernel(const __grid_constant__ LossPackParams p) {
    using T = typename Elem<F32>::type;
    extern __shared__ __align__(16) uint8_t pack_smem[];
    __shared__ float red[kPackWarps], red2[4];
    __shared__ float s_norm[128];
    __shared__ uint8_t s_valid[128];
    __shared__ int s_scan[kPackWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    launch_next();
    const bool is_w = (int)blockIdx.x < p.w_tiles;
    const int tile = is_w ? (int)blockIdx.x : (int)blockIdx.x - p.w_tiles;
    const long long row0 = (long long)tile * kLossTile;
    const long long n_rows = is_w ? p.lab.n : p.rows;

    // 2,048 chunks of 8 K slots, 4 per thread: row-major operands with neighbouring threads on
    // neighbouring chunks, the [b][k][t] layout with neighbouring threads on neighbouring rows.
    const long long t_len = is_w ? 0 : p.t_len;
    const T* src = static_cast<const T*>(is_w ? p.w : p.x);
    const bool vec = t_len == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && p.k % (F32 ? 4 : 8) == 0;
    auto item_row = [&](int i) { return t_len > 0 ? tid & 127 : i * (kPackThreads / 16) + (tid >> 4); };
    auto item_chunk = [&](int i) { return t_len > 0 ? i * (kPackThreads / 128) + (tid >> 7) : tid & 15; };
    const long long kt_base = t_len > 0 && row0 + (tid & 127) < n_rows ? x_base(row0 + (tid & 127), p.k, t_len) : 0;
    float v[kPackItems][8];
#pragma unroll
    for (int i = 0; i < kPackItems; ++i) {
        const int r = item_row(i), ch = item_chunk(i);
        const long long row = row0 + r;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row < n_rows && 8 * ch < p.k) {
            const T* a = src + (t_len > 0 ? kt_base + 8 * ch * t_len : row * p.k + 8 * ch);
            if (vec && 8 * ch + 8 <= p.k) {
                if constexpr (F32) {
                    const float4 lo = *reinterpret_cast<const float4*>(a), hi = *reinterpret_cast<const float4*>(a + 4);
                    v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = lo.z, v[i][3] = lo.w;
                    v[i][4] = hi.x, v[i][5] = hi.y, v[i][6] = hi.z, v[i][7] = hi.w;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4*>(a);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[i][2 * j] = __uint_as_float(w[j] << 16);
                        v[i][2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                }
            } else {
                const long long step = t_len > 0 ? t_len : 1;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (8 * ch + j < p.k) v[i][j] = to_f32(a[j * step]);
            }
        }
    }

    // ---- labels: which rows count, their factors, and (weight gradient) the entries with their
    // place among the warp's own of the same bin
    const int nb = 4 * p.w_tiles;                                  // 32 classes a bin
    uint16_t* counts = reinterpret_cast<uint16_t*>(pack_smem);     // [16 warps][nb]
    int* start = reinterpret_cast<int*>(pack_smem + kPackWarps * 2 * (size_t)nb);  // [nb]
    int* ents = start + nb;                                        // [128][n_top]: class << 10 | place, or -1
    if (!is_w) {
        for (int i = tid; i < kPackWarps * nb / 2; i += kPackThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0u;
        __syncthreads();
    }
    if (!is_w) {
        // lanes per row: the power of two that holds the entries (two each beyond 32)
        const int width = p.lab.n_top > 16 ? 32 : p.lab.n_top > 8 ? 16 : p.lab.n_top > 4 ? 8 : p.lab.n_top > 1 ? 4 : 1;
        const int per = min(8, 32 / width), sub = lane & (width - 1), grp = lane / width;
        const int slots = p.lab.n_top > 32 ? 2 : 1;
        uint16_t* mine = counts + (size_t)warp * nb;
        for (int r0 = 0; r0 < 8; r0 += per) {
            const int r = warp * 8 + r0 + grp;
            const long long row = row0 + r;
            const bool live = grp < per && row < p.rows;
            int c[2] = {-1, -1};
            bool bad = false;
            float g = 0.0f;
            if (live) {
                for (int s = 0; s < slots; ++s) {
                    const int e = sub + 32 * s;
                    if (e < p.lab.n_top) {
                        const int x = p.lab.target ? p.lab.target[row] : p.lab.top_idx[row * p.lab.n_top + e];
                        bad |= x >= p.lab.n;
                        if (is_class(x, p.lab.n)) {
                            const float u = p.lab.target ? 0.0f
                                                         : p.lab.top_logits[row * p.lab.n_top + e] * p.lab.inv_temp;
                            if (u != -CUDART_INF_F) c[s] = x;  // (of no share: as absent)
                        }
                    }
                }
                g = p.row_grad ? p.row_grad[row] : 1.0f;
            }
            if (bad) atomicOr(p.status + kStatusBadClass, 1);
            const uint32_t have = __ballot_sync(0xffffffffu, c[0] >= 0 || c[1] >= 0);
            const uint32_t gm = (width == 32 ? 0xffffffffu : ((1u << width) - 1u) << (grp * width));
            const bool valid = (have & gm) != 0u;
            const float f = valid ? p.lab.temp * g : 0.0f;
            if (grp < per && sub == 0) {
                s_valid[r] = valid ? 1 : 0;
                s_norm[r] = f;  // the factors, until the norms need the place
            }
            // a class named twice (rare; beyond 32 entries a lane holds two, which one match does not
            // compare)
            const uint32_t twice = __match_any_sync(0xffffffffu, c[0] >= 0 ? c[0] : ~lane) & gm;
            if (slots == 2 || __any_sync(0xffffffffu, __popc(twice) > 1)) {
                bool dup[2] = {false, false};
                for (int j = 0; j < p.lab.n_top; ++j) {
                    const int from = grp * width + (j & (width - 1));
                    const int cj = __shfl_sync(0xffffffffu, j < 32 ? c[0] : c[1], from);
#pragma unroll
                    for (int s = 0; s < 2; ++s) dup[s] |= cj >= 0 && cj == c[s] && j < sub + 32 * s;
                }
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (dup[s]) c[s] = -1;
            }
            for (int s = 0; s < slots; ++s) {
                const int e = sub + 32 * s;
                const int bin = c[s] >= 0 ? c[s] >> 5 : -1;
                const uint32_t same = __match_any_sync(0xffffffffu, bin);
                const int rank = __popc(same & ((1u << lane) - 1u));
                int at = 0;
                if (bin >= 0) {
                    at = mine[bin];
                    __syncwarp(same);
                    if (rank == 0) mine[bin] = (uint16_t)(at + __popc(same));
                }
                __syncwarp();
                if (live && e < p.lab.n_top) ents[r * p.lab.n_top + e] = c[s] >= 0 ? (c[s] << 10) | (at + rank) : -1;
            }
        }
        __syncthreads();
    }
    if (!is_w) {
        const float f = tid < 128 ? s_norm[tid] : 0.0f;
        if (F32) {
            if (tid == 0) p.tile_done[tile] = 0;
        } else {
            const int neg = __syncthreads_or(f < 0.0f);
            if (tid == 0) p.g_scale[tile] = neg ? 1.0f : 0.0f;
        }
        if (tid < 128) p.row_tab[(size_t)tile * 256 + 128 + tid] = F32 ? f : copysignf(1.0f, f);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPackItems; ++i) {
            if (row0 + item_row(i) < n_rows && !s_valid[item_row(i)]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            }
        }
    } else if (tid < 128) {
        const long long j = row0 + tid;
        p.class_e[(size_t)tile * 128 + tid] =
            j < p.lab.n ? (p.bias ? p.bias[j] * p.logit_scale : 0.0f) : -CUDART_INF_F;
    }

    // ---- scale and images
    float up = 1.0f;
    if (F32) {
        float top = 0.0f;  // of the finite values: an infinity is its own row's alone
#pragma unroll
        for (int i = 0; i < kPackItems; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[i][j]) <= CUDART_MAX_NORMAL_F ? fabsf(v[i][j]) : 0.0f);
        }
        top = warp_max(top);
        if (lane == 0) red[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPackWarps; ++i) top = fmaxf(top, red[i]);
        const int sh = shift_to(top, 14);
        up = pow2i(sh);
        if (tid == 0) (is_w ? p.w_scale : p.x_scale)[tile] = pow2i(-sh);
    } else if (p.slots) {
        // |row|: row-major operands have a row's 16 chunks in 16 neighbouring lanes, the other layout
        // has every fourth one in each of four threads; both add them up in the same tree
        float q[kPackItems];
#pragma unroll
        for (int i = 0; i < kPackItems; ++i) {
            q[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[i] = fmaf(v[i][j], v[i][j], q[i]);
        }
        if (t_len > 0) {
            float* part = reinterpret_cast<float*>(pack_smem) + p.norm_smem;  // [4][128]
            part[tid] = (q[0] + q[2]) + (q[1] + q[3]);
            __syncthreads();
            if (tid < 128) s_norm[tid] = (part[tid] + part[256 + tid]) + (part[128 + tid] + part[384 + tid]);
        } else {
#pragma unroll
            for (int i = 0; i < kPackItems; ++i) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) q[i] += __shfl_xor_sync(0xffffffffu, q[i], o);
                if ((tid & 15) == 0) s_norm[item_row(i)] = q[i];
            }
        }
        __syncthreads();
        const float norm = tid < 128 ? sqrtf(s_norm[tid]) : 0.0f;
        if (is_w) {
            const long long j = row0 + tid;
            const bool real = tid < 128 && j < p.lab.n;
            const float e = real ? (p.bias ? p.bias[j] * p.logit_scale : 0.0f) : -CUDART_INF_F;
            // (a NaN norm or bias has to survive the maximum: it then rules the bound out)
            const float wn = warp_max(norm), we = warp_max(e);
            const int bad = __syncthreads_or(real && (isnan(norm) || isnan(e)));
            if (lane == 0 && warp < 4) {
                red[warp] = wn;
                red2[warp] = we;
            }
            __syncthreads();
            if (tid == 0)
                p.w_bound[tile] = make_float2(bad ? CUDART_NAN_F : fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])),
                                              fmaxf(fmaxf(red2[0], red2[1]), fmaxf(red2[2], red2[3])));
        } else if (tid < 128) {
            p.x_norm[(size_t)tile * 128 + tid] = norm;
        }
    }
    uint8_t* img = (is_w ? p.w_img : p.x_img) + (size_t)tile * (F32 ? 2 * kLossImage : kLossImage);
#pragma unroll
    for (int i = 0; i < kPackItems; ++i) {
        const uint32_t off = image_chunk(item_row(i), item_chunk(i));
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (F32) {
                const float a = v[i][2 * j] * up, b = v[i][2 * j + 1] * up;
                const __half2 hv = __floats2half2_rn(a, b);
                const float2 hf = __half22float2(hv);
                const __half2 lv = __floats2half2_rn(a - hf.x, b - hf.y);
                h[j] = *reinterpret_cast<const uint32_t*>(&hv);
                l[j] = *reinterpret_cast<const uint32_t*>(&lv);
            } else {
                const __nv_bfloat162 hv = __floats2bfloat162_rn(v[i][2 * j], v[i][2 * j + 1]);
                h[j] = *reinterpret_cast<const uint32_t*>(&hv);
            }
        }
        *reinterpret_cast<uint4*>(img + off) = make_uint4(h[0], h[1], h[2], h[3]);
        if constexpr (F32) *reinterpret_cast<uint4*>(img + kLossImage + off) = make_uint4(l[0], l[1], l[2], l[3]);
    }
    if (!F32 && p.slots) {
        // the bias (natural units) in three bf16 parts, against ones in the features: the parts'
        // products with 1 are exact, so a score carries its bias to 24 bits. Padding classes: -inf.
        __syncthreads();  // the chunks that hold the slots are written above, by other threads
        if (tid < 128) {
            float rest = row0 + tid < p.lab.n ? (is_w && p.bias ? p.bias[row0 + tid] : 0.0f) : -CUDART_INF_F;
            for (int part = 0; part < 3; ++part) {
                const __nv_bfloat16 here = __float2bfloat16_rn(is_w ? rest : 1.0f);
                rest = isfinite(__bfloat162float(here)) ? rest - __bfloat162float(here) : 0.0f;
                const int kk = p.k + part;
                *reinterpret_cast<__nv_bfloat16*>(img + image_chunk(tid, kk >> 3) + 2 * (kk & 7)) = here;
            }
        }
    }
    if (is_w) return;

    // ---- the entries' places: counts -> each warp's first position within its bin, bins' starts
    const int per = (nb + kPackThreads - 1) / kPackThreads, b0 = tid * per, b1 = min(nb, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        int tot = 0;
        for (int w = 0; w < kPackWarps; ++w) {
            const int c = counts[(size_t)w * nb + b];
            counts[(size_t)w * nb + b] = (uint16_t)tot;
            tot += c;
        }
        start[b] = sum;
        sum += tot;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += s_scan[w];
    int2* range = p.sp_off + (size_t)tile * nb;
    for (int b = b0; b < b1; ++b) {
        const int next = b + 1 < b1 ? start[b + 1] : sum;
        range[b] = make_int2(base + start[b], base + next);
    }
    for (int b = b0; b < b1; ++b) start[b] += base;
    __syncthreads();
    int2* out = p.sp_ent + (size_t)tile * 128 * p.lab.n_top;
    const int live = (int)min((long long)128, p.rows - row0) * p.lab.n_top;
    for (int i = tid; i < live; i += kPackThreads) {
        const int e = ents[i];
        int at = -1;
        if (e >= 0) {
            const int r = i / p.lab.n_top, c = e >> 10, bin = c >> 5;
            at = start[bin] + counts[(size_t)(r >> 3) * nb + bin] + (e & 1023);
            out[at].x = (r << 5) | (c & 31);
        }
        p.sp_pos[(size_t)tile * 128 * p.lab.n_top + i] = at;
    }
}

// ------------------------------------------------------------------------------- main pass
namespace {

// Warps: 0 producer, 1 issuer of the scores (and TMEM), 2 issuer of the second products, 3 idle; four
// softmax warpgroups (warps 4-19): two for the even and two for the odd streamed tiles, 64 columns
// each; two adding warpgroups (20-27), 64 features of the second products each.
// Softmax and adding are apart so that a softmax warpgroup goes on to its next tile without waiting
// for the tensor core to use its last. Two issuers, because the tensor core queues only a few
// instructions: while one waits on its barriers the other's products run (with one issuer, its waits
// and the products add up).
// Scores live in buffers of 128 TMEM columns: two in f32, whose own operand (hi | lo) takes 128
// columns; three in bf16, whose own operand stays in shared memory, so that the next scores are there
// when a softmax warpgroup comes for them. (An operand in TMEM costs the tensor core less
// shared-memory bandwidth; f32 is bound by the tensor core, bf16 is not. Buffers of half a tile's
// scores are no way out: an instruction of 64 columns takes as long as one of 128.)
constexpr int kMainThreads = 896;
constexpr int kLaunchRegs = 72;  // 65,536 registers / 896 threads
constexpr int kCtrlRegs = 40, kSoftRegs = 72, kAddRegs = 88;
// What the producer and issuers give back has to cover what the adding warps take: their setmaxnreg
// waits for it, without a limit. `launch`: registers a thread that a variant was built with, which the
// softmax warps keep; loss_kernel_setup checks it for each.
constexpr bool split_fits(int launch) { return 128 * (launch - kCtrlRegs) >= 256 * (kAddRegs - launch); }
static_assert(kSoftRegs == kLaunchRegs && split_fits(kLaunchRegs) && !split_fits(kLaunchRegs - 8), "register split");
static_assert(kMainThreads * kLaunchRegs <= 65536, "registers of an SM");

template <bool F32>
struct Ring {
    static constexpr uint32_t kStage = F32 ? 2u * kLossImage : kLossImage;
    static constexpr uint32_t kStages = F32 ? 3u : 4u;
    static constexpr uint32_t kTab = kStage * kStages;              // column tables, 1 KB a stage
    static constexpr uint32_t kOwn = kTab + 1024u * kStages;        // bf16: two images of the own operand
    static constexpr uint32_t kEnd = kOwn + (F32 ? 0u : 2u * kLossImage);
    static constexpr uint32_t kBufs = F32 ? 2u : 3u;                // score buffers of 128 TMEM columns
    static constexpr uint32_t kTS = F32 ? 128u : 0u;                // their first column (f32: after the own operand)
};
constexpr uint32_t kMOffBars = 200704;             // after the stages, their column tables and own images
constexpr uint32_t kMOffMisc = kMOffBars + 512;   // [0] TMEM base, [1] abort flag
constexpr uint32_t kMOffMs = kMOffMisc + 64;      // [4][128] float2: the softmax warpgroups' row state
constexpr uint32_t kMOffUnion = kMOffMs + 4096;
constexpr uint32_t kMOffRing = kMOffUnion;         // row pass: [4 tiles][128] f32, offset of a tile's probabilities
constexpr uint32_t kMOffTop = kMOffUnion + 2048;   // row pass: [2][4][128] f32, maxima of a tile's two halves
constexpr uint32_t kMOffNamed = kMOffTop + 4096;   // row pass: [16 warps][32 rows][2] bits of the named columns
constexpr uint32_t kPatchRow = 12;                 // floats per class row of a label patch (8 used:
                                                   // the 16-byte rows then fall on distinct banks)
constexpr uint32_t kMOffPatch = kMOffUnion;        // weight pass: [16 warps][32][kPatchRow] f32
constexpr uint32_t kMSmemUsed = kMOffPatch + 16 * 32 * kPatchRow * 4;
constexpr uint32_t kMSmemBytes = kMSmemUsed + 1024;
static_assert(Ring<true>::kEnd <= kMOffBars && Ring<false>::kEnd <= kMOffBars && Ring<false>::kOwn % 1024 == 0,
              "shared memory map");
static_assert(kMSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(kMOffNamed + 16 * 64 * 4 <= kMSmemUsed, "row pass within the union");

constexpr int kLBarFull = 0;               // [4] tile and column table landed
constexpr int kLBarEmpty = 4;              // [4] the tile's products done, its softmax warps done with the table
constexpr int kLBarAFull = 8;              // [2] own operand in place (f32: [0] only)
constexpr int kLBarAEmpty = 10;            // [2] the unit's products done with it
constexpr int kLBarSFull = 12;             // [3] scores of a buffer in TMEM
constexpr int kLBarPFull = 15;             // [3][2 halves] its probabilities in their place
constexpr int kLBarOFull = 21;             // the tile's second product in TMEM
constexpr int kLBarOEmpty = 22;            // added up, the buffer free
constexpr int kLBarRing = 23;              // [4] a tile's offsets written
constexpr int kLBarMsFull = 27;            // row states of a unit written
constexpr int kLBarMsEmpty = 28;           // and read
constexpr int kLBarTop = 29;               // [2 parities][4 quadrants] both halves' maxima written
constexpr int kLBarSFree = 37;             // [3] a buffer's probabilities used up: it may take scores again
constexpr int kLBarDone = 40;              // [2 issuers] every product retired (teardown)
static_assert(8 * (kLBarDone + 2) <= 512, "barrier area");

// TMEM columns: f32 own operand from 0, score buffers (Ring), second product
constexpr uint32_t kTOwn = 0, kTO = 384;
static_assert(Ring<true>::kTS + 128 * Ring<true>::kBufs <= kTO && Ring<false>::kTS + 128 * Ring<false>::kBufs <= kTO,
              "TMEM columns");
constexpr uint32_t kLSleepNs = 20000;

struct Waiter {
    volatile uint32_t* abort_flag;
    int* status;
    unsigned long long timeout_ns;
};

// Bounded wait: gives up when another role has, or after the time limit (device status set);
// every role then leaves its loop and the kernel ends normally.
__device__ __forceinline__ bool loss_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                               int* status, unsigned long long timeout_ns, int where) {
    const uint64_t t0 = globaltimer_ns();
    while (true) {
        if (mbar_try_wait_sleep(bar, parity, kLSleepNs)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > timeout_ns) {
            *abort_flag = 1u;
            atomicOr(status, kDevTimeout);
            atomicExch(status + 1, where);
            return false;
        }
    }
}
// The issuers' waits poll a while before they sleep (their wake-up is on every tile's critical path)
// and look at all the barriers they need at once.
__device__ __forceinline__ bool issuer_wait(uint32_t bar, uint32_t parity, const Waiter& w, int where) {
    bool ok = false;
    for (int i = 0; i < 64 && !ok; ++i) ok = mbar_try_wait(bar, parity);
    if (!ok) ok = loss_wait_slow(bar, parity, w.abort_flag, w.status, w.timeout_ns, where);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool issuer_wait2(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1,
                                             const Waiter& w, int where) {
    bool ok = false;
    for (int i = 0; i < 64 && !ok; ++i) ok = mbar_try_wait2(bar0, parity0, bar1, parity1);
    if (!ok)
        ok = loss_wait_slow(bar0, parity0, w.abort_flag, w.status, w.timeout_ns, where) &&
             loss_wait_slow(bar1, parity1, w.abort_flag, w.status, w.timeout_ns, where + 20);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool issuer_wait3(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1,
                                             uint32_t bar2, uint32_t parity2, const Waiter& w, int where) {
    bool ok = false;
    for (int i = 0; i < 64 && !ok; ++i) ok = mbar_try_wait3(bar0, parity0, bar1, parity1, bar2, parity2);
    if (!ok)
        ok = loss_wait_slow(bar0, parity0, w.abort_flag, w.status, w.timeout_ns, where) &&
             loss_wait_slow(bar1, parity1, w.abort_flag, w.status, w.timeout_ns, where) &&
             loss_wait_slow(bar2, parity2, w.abort_flag, w.status, w.timeout_ns, where + 20);
    return __all_sync(0xffffffffu, ok);
}
// Uniform over the (converged) warp.
__device__ __forceinline__ bool loss_wait(uint32_t bar, uint32_t parity, const Waiter& w, int where) {
    bool ok = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (!ok) ok = loss_wait_slow(bar, parity, w.abort_flag, w.status, w.timeout_ns, where);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void loss_drain(uint32_t bar, uint32_t parity, const Waiter& w) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait_sleep(bar, parity, kLSleepNs)) {
        if (globaltimer_ns() - t0 > w.timeout_ns) {
            atomicOr(w.status, kDevTimeout);
            return;
        }
    }
}

struct LUnit {
    int own, c0, c1;
};
// The unit that this CTA takes in wave k, or -1: CTA b takes unit b of every full wave, and unit
// grid - 1 - b of a last one that is not full. The first units are so those of the CTAs with a unit
// less: in the weight pass they hold class 0, the blank, whose tile has most rows' labels and takes
// up to 1.6 times as long as the others (18,710 classes: 4 x 147 units, CTAs 0-3 have three).
__device__ __forceinline__ int lunit_at(int k, const LossMainParams& p) {
    const int units = p.whole_units + (p.own_tiles - p.whole_units) * p.n_splits;
    const int base = k * (int)gridDim.x, b = (int)blockIdx.x;
    const int u = base + (int)gridDim.x <= units ? base + b : base + (int)gridDim.x - 1 - b;
    return u < units ? u : -1;
}
__device__ __forceinline__ LUnit lunit(int u, const LossMainParams& p) {
    if (u < p.whole_units) return {u, 0, p.str_tiles};
    const int v = u - p.whole_units, b = v / p.n_splits, s = v - b * p.n_splits;
    const int c0 = s * p.tiles_per_split;
    return {p.whole_units + b, c0, min(c0 + p.tiles_per_split, p.str_tiles)};
}

// 16 columns' values (8 pairs) as 16-bit tensor-core operands, over the 16 score columns they come
// from: f32 as fp16 hi (8 columns) and lo (8 columns), whose sum holds ~22 bits and whose products
// are exact in the f32 accumulator; bf16 by one rounding (half a step of the operand type, as the
// features' own), or with TWO as hi and lo in the same places, whose sum is 2^-16 off at most.
template <bool F32, bool TWO = false>
__device__ __forceinline__ void store_probs(uint32_t taddr, const float2 (&g)[8]) {
    if constexpr (F32) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __half2 h = __floats2half2_rn(g[i].x, g[i].y);
            const float2 hf = __half22float2(h);
            const float2 d = __fadd2_rn(g[i], make_float2(-hf.x, -hf.y));
            const __half2 l = __floats2half2_rn(d.x, d.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
            w[8 + i] = *reinterpret_cast<const uint32_t*>(&l);
        }
        tmem_st32x32b_x16(taddr, w);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(g[i].x, g[i].y);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st32x32b_x8(taddr, w);
        if constexpr (TWO) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // a bf16 is the upper half of the f32 of the same value
                const float2 d = __fadd2_rn(g[i], make_float2(-__uint_as_float(w[i] << 16),
                                                              -__uint_as_float(w[i] & 0xffff0000u)));
                const __nv_bfloat162 l = __floats2bfloat162_rn(d.x, d.y);
                w[i] = *reinterpret_cast<const uint32_t*>(&l);
            }
            tmem_st32x32b_x8(taddr + 8u, w);
        }
    }
}

// The labels of a warp's 32 classes in a tile (weight pass), a window of 32 at a time, rows
// ascending: each lane holds one entry of the current window and, where the list goes on, one of the
// next, in flight meanwhile.
struct LabelWindow {
    int2 e, n;        // (row << 5 | class, gradient)
    int next, end;    // first entry after the current window
    uint32_t groups;  // groups of 8 of this half's rows that have an entry in the window
    int last;         // group of the window's last entry where entries follow it, else beyond any group
    int group;        // group of this lane's entry; outside 0..7: none, or in the other half
};
constexpr int kNoLabel = 0x7fffffff;
constexpr int kNoPatch = -1;  // a patch cell without an entry: bits that no computed value has
// The labels of a warp's 64 columns in a tile (row pass): entries of two runs of 32 classes, one after
// the other.
struct NamedRange {
    int next, mid, end;  // first entry, first of the second 32 classes, end
    int e;               // this lane's of the first 32 entries: row << 5 | class within its 32
};
__device__ __forceinline__ int named_entry(const int2* ent, int i, int end) {
    return i < end ? chain_load(&ent[i].x) : kNoLabel;
}
__device__ __forceinline__ int2 window_entry(const LabelWindow& w, const int2* ent, int lane) {
    return w.next + lane < w.end ? chain_load(ent + w.next + lane) : make_int2(kNoLabel, 0);
}
__device__ __forceinline__ void window_use(LabelWindow& w, const int2* ent, int lane, int half) {
    w.next += 32;
    w.group = (w.e.x >> 8) - 8 * half;
    w.groups = __reduce_or_sync(0xffffffffu, (uint32_t)w.group < 8u ? 1u << w.group : 0u);
    w.last = 8;
    if (w.next < w.end) {
        w.n = window_entry(w, ent, lane);
        w.last = __shfl_sync(0xffffffffu, w.group, 31);
    }
}

}  // namespace

// Streamed tiles whose second products the tensor core adds up before the adding warps do.
// The tensor core's f32 accumulator rounds toward zero, a bias of up to 2^-24 of the sum a step. In
// f32 every tile's product is added in registers: 24 steps stay below the operands' own error. In
// bf16 the 8 steps of 32 tiles leave at most 2^-16, a hundredth of the probabilities' rounding; that
// takes the adding off every tile's path, where the offset does not move (the weight pass; the row
// pass where every row of the own tile is bounded, see below).
constexpr int kAddEvery = 32;
// bf16 passes over at most this many streamed tiles: the probabilities in two parts, for a second run
// of 8 instructions a tile. Sums of few terms do not average their rounding away: with one part dw of 3
// to 8 rows and da over 87 classes were off by 1.5 to 1.9 times their own type's rounding, of 128 or
// more rows or classes mostly by 1.3 times, with two parts by that rounding alone. (A class that few
// rows name has few large terms in a long step too, and keeps the one rounding there: 2^-9 of each
// term, as of any gradient that enters a bf16 product.)
// Above it one rounding does: of 122,880 rows, gradients lie as near float64 as f32 arithmetic's rounded
// once (1.8e-3 both). A variant of its own (TWO): a test inside the kernel alone slowed long steps down.
constexpr int kTwoPartTiles = 8;

// Units (own tile, range of streamed tiles), persistent over the grid. Per streamed tile: scores
// S = own . tile^T (tensor core), a softmax warpgroup turns them into
// probabilities (row pass: against the running maximum, the classes that the row names left out;
// weight pass: 2^(s - lse) times the rows' gradient factors, the labels' gradients in their place) in
// the same TMEM columns, and a second product O = P . tile reads the same tile the other way round;
// the adding warps sum it in registers.
// f32: three products each (hi.lo, lo.hi, hi.hi).
// bf16 with slots: the scores come with their bias, so they need no column table in the row pass;
// and as bf16 probabilities have f32's range, a row's offset need not follow its maximum: by
// Cauchy-Schwarz every logit lies within |x_r| max|w| of the largest bias, so where that leaves a
// spread of at most 80 binary orders the upper bound itself is the offset, every probability is at
// most 1, and what underflows (below 2^-126) is 2^-46 of the largest. Rows beyond it (a warp at a
// time) follow the running maximum as the others do.
template <bool F32, bool WPASS, bool SLOTS, bool TWO = false>
__global__ void __launch_bounds__(kMainThreads, 1) loss_main_kernel(const __grid_constant__ LossMainParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    uint32_t* misc = reinterpret_cast<uint32_t*>(gbase + kMOffMisc);
    constexpr uint32_t kStage = Ring<F32>::kStage, kStages = Ring<F32>::kStages;
    constexpr uint32_t kTabBytes = WPASS ? 1024u : 512u;
    auto bar = [&](int i) -> uint32_t { return base + kMOffBars + 8u * (uint32_t)i; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Waiter wt{misc + 1, p.status, p.timeout_ns};
    const bool with_o = WPASS || p.part_o != nullptr;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 4; ++s) {
            mbar_init(bar(kLBarFull + s), 1);
            mbar_init(bar(kLBarEmpty + s), 9);  // the product's commit, eight warps
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(kLBarAFull + i), F32 ? 512 : 1);  // bf16: one bulk copy
            mbar_init(bar(kLBarAEmpty + i), 1);
        }
        for (int i = 0; i < 3; ++i) {
            mbar_init(bar(kLBarSFull + i), 1);
            mbar_init(bar(kLBarSFree + i), 1);
            mbar_init(bar(kLBarPFull + 2 * i), 4);
            mbar_init(bar(kLBarPFull + 2 * i + 1), 4);
        }
        mbar_init(bar(kLBarOFull), 1);
        mbar_init(bar(kLBarOEmpty), 8);
        for (int i = 0; i < 4; ++i) mbar_init(bar(kLBarRing + i), 4);
        mbar_init(bar(kLBarMsFull), 512);
        for (int i = 0; i < 8; ++i) mbar_init(bar(kLBarTop + i), 2);
        mbar_init(bar(kLBarMsEmpty), 128);
        mbar_init(bar(kLBarDone), 1);
        mbar_init(bar(kLBarDone + 1), 1);
        misc[1] = 0u;
        fence_mbar_init();
    }
    for (uint32_t i = threadIdx.x; i < 16 * 32 * kPatchRow; i += kMainThreads)
        reinterpret_cast<int*>(gbase + kMOffPatch)[i] = WPASS ? kNoPatch : 0;
    if (warp == 1) {
        tmem_alloc(base + kMOffMisc, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    const int feat = 16 * p.ksteps;
    launch_next();
    wait_previous();
    // slots, row pass: the reach of a row's logits around the largest bias is |x_r| max|w|
    float w_max = 0.0f, e_max = -CUDART_INF_F;
    if (SLOTS && !WPASS && warp >= 2) {
        bool nan = false;
        for (int t = lane; t < p.str_tiles; t += 32) {
            const float2 b = chain_load(p.w_bound + t);
            nan |= isnan(b.x);
            w_max = fmaxf(w_max, b.x);
            e_max = fmaxf(e_max, b.y);
        }
        w_max = warp_max(w_max);
        e_max = warp_max(e_max);
        if (__any_sync(0xffffffffu, nan)) w_max = CUDART_INF_F;
    }
    auto reach_of = [&](int own, int row) {
        return p.logit_scale * chain_load(p.x_norm + (size_t)own * 128 + row) * w_max * 1.001f;
    };
    auto in_bounds = [&](float reach) { return reach <= 40.0f && fabsf(reach + e_max) < 1e6f; };
    // tiles added up in TMEM at a time, for this own tile (every role that asks finds the same)
    auto add_every = [&](int own) -> int {
        if (F32) return 1;
        if (WPASS) return kAddEvery;
        if (!SLOTS) return 1;
        bool all = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) all = all && in_bounds(reach_of(own, 32 * i + lane));
        return __all_sync(0xffffffffu, all) ? kAddEvery : 1;
    };

    if (warp < 4) {
        setmaxnreg_dec<kCtrlRegs>();
        if (warp == 0) {
            // ------------------------------------------------------------ producer
            uint32_t cc = 0, issued = 0, uc = 0, owns = 0;
            bool ok = true;
            for (int u; ok && (u = lunit_at((int)uc, p)) >= 0; ++uc) {
                const LUnit U = lunit(u, p);
                if (!F32) {  // the unit's own image, in the slot that the unit before the last has left
                    const uint32_t w = uc & 1u;
                    ok = loss_wait(bar(kLBarAEmpty + w), ((uc >> 1) & 1u) ^ 1u, wt, 114);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar(kLBarAFull + w), kLossImage);
                        bulk_copy_g2s(base + Ring<F32>::kOwn + w * kLossImage, p.own + (size_t)U.own * kLossImage,
                                      kLossImage, bar(kLBarAFull + w));
                    }
                    __syncwarp();
                    owns = uc + 1;
                }
                for (int c = U.c0; c < U.c1; ++c, ++cc) {
                    const uint32_t s = cc % kStages;
                    ok = loss_wait(bar(kLBarEmpty + s), ((cc / kStages) & 1u) ^ 1u, wt, 101);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar(kLBarFull + s), kStage + kTabBytes);
                        bulk_copy_g2s(base + s * kStage, p.str + (size_t)c * kStage, kStage, bar(kLBarFull + s));
                        bulk_copy_g2s(base + Ring<F32>::kTab + s * 1024u, p.col_tab + (size_t)c * (kTabBytes / 4),
                                      kTabBytes, bar(kLBarFull + s));
                    }
                    __syncwarp();
                    issued = cc + 1;
                }
            }
            // no copy outlives the CTA
            for (uint32_t s = 0; s < kStages && s < issued; ++s)
                loss_drain(bar(kLBarFull + s), ((issued - 1 - s) / kStages) & 1u, wt);
            for (uint32_t w = 0; w < 2 && w < owns; ++w) loss_drain(bar(kLBarAFull + w), ((owns - 1 - w) / 2) & 1u, wt);
        } else if (warp == 1) {
            // ------------------------------------------------------------ issuer of the scores
            // Ring positions advance by increments: the issuers are the tensor core's only feed.
            const uint32_t id_s = idesc_16b(!F32, false, 128, 128);
            const uint64_t k_desc = smem_desc_k_sw128(base);
            uint32_t st = 0, sph = 0, b = 0, fph = 1, uc = 0;  // stage, buffer, their phases (the buffer: freed)
            bool ok = true;
            for (int u; ok && (u = lunit_at((int)uc, p)) >= 0; ++uc) {
                const LUnit U = lunit(u, p);
                const uint32_t w = F32 ? 0u : uc & 1u;
                ok = issuer_wait(bar(kLBarAFull + w), F32 ? uc & 1u : (uc >> 1) & 1u, wt, 103);
                const uint64_t own_desc = k_desc + ((Ring<F32>::kOwn + w * kLossImage) >> 4);
                for (int c = U.c0; ok && c < U.c1; ++c) {
                    ok = issuer_wait2(bar(kLBarFull + st), sph, bar(kLBarSFree + b), fph, wt, 102);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t b_desc = k_desc + st * (uint64_t)(kStage >> 4);
                    const uint32_t d = tmem + Ring<F32>::kTS + 128u * b;
                    if (F32)
                        mma_scores_f32_warp(d, tmem + kTOwn, b_desc, id_s, p.ksteps);
                    else
                        mma_scores_bf16_warp(d, own_desc, b_desc, id_s, p.ksteps);
                    mma_commit_warp(bar(kLBarSFull + (int)b));
                    if (++st == kStages) st = 0u, sph ^= 1u;
                    if (++b == Ring<F32>::kBufs) b = 0u, fph ^= 1u;
                }
                if (!ok) break;
                mma_commit_warp(bar(kLBarAEmpty + w));
            }
            mma_commit_warp(bar(kLBarDone));
            loss_drain(bar(kLBarDone), 0u, wt);
        } else if (warp == 2) {
            // -------------------------------------------------- issuer of the second products
            const uint32_t id_o = idesc_16b(!F32, true, 128, (uint32_t)feat);
            const uint64_t mn_desc = smem_desc_mn_sw128(base);
            uint32_t st = 0, b = 0, pph = 0, oph = 1;  // stage, buffer and phase of its probabilities; O's release
            bool ok = true;
            for (int k = 0, u; ok && (u = lunit_at(k, p)) >= 0; ++k) {
                const LUnit U = lunit(u, p);
                const int every = with_o ? add_every(U.own) : 1;
                int held = 0;  // products in O so far
                for (int c = U.c0; ok && c < U.c1; ++c) {
                    // both halves' probabilities, and what O held added up
                    ok = issuer_wait3(bar(kLBarPFull + 2 * (int)b), pph, bar(kLBarPFull + 2 * (int)b + 1), pph,
                                      bar(kLBarOEmpty), with_o ? oph : 1u, wt, 104);
                    if (!ok) break;
                    tc_fence_after();
                    if (with_o) {
                        const uint64_t b_desc = mn_desc + st * (uint64_t)(kStage >> 4);
                        const uint32_t a = tmem + Ring<F32>::kTS + 128u * b;
                        if (F32)
                            mma_rows_f32_warp(tmem + kTO, a, b_desc, id_o);
                        else
                            mma_rows_bf16_warp(tmem + kTO, a, b_desc, id_o, held > 0 ? 1u : 0u);
                        if (TWO) mma_rows_bf16_warp(tmem + kTO, a + 8u, b_desc, id_o, 1u);
                        if (++held == every || c + 1 == U.c1) {
                            mma_commit_warp(bar(kLBarOFull));
                            oph ^= 1u;
                            held = 0;
                        }
                    }
                    mma_commit_warp(bar(kLBarSFree + (int)b));
                    mma_commit_warp(bar(kLBarEmpty + (int)st));
                    if (++st == kStages) st = 0u;
                    if (++b == Ring<F32>::kBufs) b = 0u, pph ^= 1u;
                }
            }
            mma_commit_warp(bar(kLBarDone + 1));
            loss_drain(bar(kLBarDone + 1), 0u, wt);
        }
    } else if (warp < 20) {
        // (kSoftRegs is what the kernel was launched with)
        // ------------------------------------------------------------- softmax warpgroups
        const uint32_t wg = (uint32_t)(warp - 4) >> 2, g = wg >> 1, half = wg & 1u;
        const int quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t patch = base + kMOffPatch + (uint32_t)(warp - 4) * 32u * kPatchRow * 4u;
        const uint32_t t_bufs = tmem + lanes + Ring<F32>::kTS + 64u * half;
        float* ring = reinterpret_cast<float*>(gbase + kMOffRing);
        volatile float* tops = reinterpret_cast<volatile float*>(gbase + kMOffTop);
        // tiles, units, tiles whose offsets were handed on, tiles whose maximum was exchanged
        uint32_t cc = 0, uc = 0, rc = 0, tc = 0;
        bool ok = true;
        for (int u; ok && (u = lunit_at((int)uc, p)) >= 0; ++uc) {
            const LUnit U = lunit(u, p);
            const uint32_t n = (uint32_t)(U.c1 - U.c0);
            // This pair of warpgroups takes every tile whose number in the CTA's whole sequence has its
            // parity. Scores come in that order, so the phase before the one it waits for is over (a wait
            // on a phase's parity is good only then), however units of odd length shift the buffers.
            const uint32_t i0 = (g ^ cc) & 1u;
            // labels of the first of them (weight pass): range, then entries
            LabelWindow lw{};
            const int2* ranges = p.sp_off + (size_t)(U.c0 + (int)i0) * 4 * p.own_tiles + 4 * U.own + quad;
            const int2* ent = p.sp_ent + (size_t)(U.c0 + (int)i0) * 128 * p.n_top;
            if (WPASS && i0 < n) {
                const int2 first = chain_load(ranges);
                lw.next = first.x;
                lw.end = first.y;
                lw.e = window_entry(lw, ent, lane);
            }
            // the same for the row pass: which of its columns the warp's rows name
            NamedRange nr{};
            const int4* named = reinterpret_cast<const int4*>(p.sp_off + (size_t)U.own * 4 * p.str_tiles +
                                                              4 * (U.c0 + (int)i0) + 2 * (int)half);
            const int2* named_ent = p.sp_ent + (size_t)U.own * 128 * p.n_top;
            uint32_t* bits = reinterpret_cast<uint32_t*>(gbase + kMOffNamed) + (warp - 4) * 64;
            if (!WPASS && i0 < n) {
                const int4 first = chain_load(named);
                nr = {first.x, first.y, first.w, named_entry(named_ent, first.x + lane, first.w)};
            }
            if (F32) {
                // own operand -> TMEM: warpgroup wg takes K slots 64 half .. 64 half + 63 of the lane's
                // row, of the high part (even tiles' warpgroups) or the low part (odd)
                ok = loss_wait(bar(kLBarAEmpty), (uc & 1u) ^ 1u, wt, 106);
                if (!ok) break;
                tc_fence_after();
                if ((int)(4 * half) < p.ksteps) {
                    const uint8_t* img = p.own + (size_t)U.own * kStage + g * kLossImage;
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint4 x = chain_load(reinterpret_cast<const uint4*>(img + image_chunk(r, 8 * half + j)));
                        w[4 * j] = x.x, w[4 * j + 1] = x.y, w[4 * j + 2] = x.z, w[4 * j + 3] = x.w;
                    }
                    tmem_st32x32b_x32(tmem + lanes + kTOwn + 64u * g + 32u * half, w);
                    tmem_st_wait();
                }
                tc_fence_before();
                mbar_arrive(bar(kLBarAFull));
            }

            const float own_mul = F32 ? p.logit_scale * chain_load(p.own_scale + U.own) : p.logit_scale;
            const float lane_e = WPASS && !SLOTS ? chain_load(p.lane_e + (size_t)U.own * 128 + r) : 0.0f;
            // the tiles' offsets go to the adding warps only where they move
            const bool ringed = !WPASS && with_o && add_every(U.own) == 1;
            bool bounded = false;
            float upper = 0.0f;
            if (SLOTS && !WPASS) {
                const float reach = reach_of(U.own, r);
                upper = reach + e_max;
                bounded = __all_sync(0xffffffffu, in_bounds(reach));
            }
            float off = -CUDART_INF_F, sum = 0.0f, carry = 0.0f;  // weight pass: sum + carry = bias gradient
            for (uint32_t i = i0; i < n; i += 2) {
                const int c = U.c0 + (int)i;
                const uint32_t s = (cc + i) % kStages;
                const uint32_t tab = base + Ring<F32>::kTab + s * 1024u + 256u * half;
                const float str_s = F32 ? chain_load(p.str_scale + c) : 1.0f;
                const float gs = WPASS ? chain_load(p.g_scale + c) : 1.0f;
                // the next tile's label range is fetched under this tile, its entries at this tile's end
                int2 next_range = make_int2(0, 0);
                if (WPASS) {
                    ranges += 8 * p.own_tiles;
                    if (i + 2 < n) next_range = chain_load(ranges);
                }
                int4 next_named = make_int4(0, 0, 0, 0);
                if (!WPASS) {
                    named += 4;
                    if (i + 2 < n) next_named = chain_load(named);
                }
                // (not below the least normal: a named column's -inf must stay one)
                const float mul1 = fmaxf(own_mul * str_s, 1.17549435e-38f);
                const float2 mul = make_float2(mul1, mul1);
                // the named columns of the warp's rows, a row a lane: their scores become -inf.
                // Gathered while the scores are on their way.
                uint32_t bits0 = 0, bits1 = 0, chunks = 0;
                if (!WPASS && nr.next < nr.end) {
                    bool hit = false;
                    for (int at = nr.next; at < nr.end; at += 32) {
                        if (at != nr.next) nr.e = named_entry(named_ent, at + lane, nr.end);
                        if (nr.e >> 10 == quad) {
                            atomicOr(bits + ((nr.e >> 5) & 31) * 2 + (at + lane >= nr.mid ? 1 : 0), 1u << (nr.e & 31));
                            hit = true;
                        }
                    }
                    if (__any_sync(0xffffffffu, hit)) {
                        __syncwarp();
                        bits0 = bits[2 * lane];
                        bits1 = bits[2 * lane + 1];
                        bits[2 * lane] = bits[2 * lane + 1] = 0u;
                        const uint32_t all0 = __reduce_or_sync(0xffffffffu, bits0);
                        const uint32_t all1 = __reduce_or_sync(0xffffffffu, bits1);
                        chunks = ((all0 & 0xffffu) ? 1u : 0u) | ((all0 >> 16) ? 2u : 0u) |
                                 ((all1 & 0xffffu) ? 4u : 0u) | ((all1 >> 16) ? 8u : 0u);
                    }
                }
                const uint32_t buf = (cc + i) % Ring<F32>::kBufs;
                const uint32_t t_s = t_bufs + 128u * buf;
                ok = loss_wait(bar(kLBarSFull + (int)buf), ((cc + i) / Ring<F32>::kBufs) & 1u, wt, 107);
                // the column table came with the tile: its barrier has passed, but this warp has to
                // observe it before it reads what the copy wrote
                ok = ok && loss_wait(bar(kLBarFull + s), ((cc + i) / kStages) & 1u, wt, 108);
                if (!ok) break;
                tc_fence_after();
                // (a chunk of 16 columns in which no row of the warp names one passes by)
                auto drop_named = [&](uint32_t (&x)[16], int q) {
                    if ((chunks >> q) & 1u) {
                        const uint32_t here = (q < 2 ? bits0 : bits1) >> (16 * (q & 1));
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if ((here >> j) & 1u) x[j] = 0xff800000u;
                    }
                };
                if (SLOTS && !WPASS && bounded) {
                    off = upper;
                    if (with_o && half == 0 && ringed) ring[((rc + i) & 3u) * 128 + r] = off;
                    const float2 sub2 = make_float2(-off, -off);
                    float2 ts = make_float2(0.f, 0.f);
#pragma unroll (F32 ? 1 : 4)
                    for (int q = 0; q < 4; ++q) {
                        uint32_t x[16];
                        tmem_ld32x32b_x16(t_s + 16u * q, x);
                        tmem_ld_wait16(x);
                        drop_named(x, q);
                        float2 pr[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 a = __ffma2_rn(as_pair(x[2 * j], x[2 * j + 1]), mul, sub2);
                            pr[j] = make_float2(ex2_approx(a.x), ex2_approx(a.y));
                            ts = __fadd2_rn(ts, pr[j]);
                        }
                        if (with_o) store_probs<F32, TWO>(t_s + 16u * q, pr);
                    }
                    sum += ts.x + ts.y;
                } else if constexpr (!WPASS) {
                    float top = -CUDART_INF_F;
#pragma unroll (F32 ? 1 : 4)
                    for (int q = 0; q < 4; ++q) {
                        uint32_t x[16];
                        tmem_ld32x32b_x16(t_s + 16u * q, x);
                        tmem_ld_wait16(x);
                        drop_named(x, q);
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 e = SLOTS ? make_float4(0.f, 0.f, 0.f, 0.f) : lds128(tab + 4u * (16 * q + j));
                            const float2 a = __ffma2_rn(as_pair(x[j], x[j + 1]), mul, make_float2(e.x, e.y));
                            const float2 b = __ffma2_rn(as_pair(x[j + 2], x[j + 3]), mul, make_float2(e.z, e.w));
                            top = max3f(top, a.x, a.y);
                            top = max3f(top, b.x, b.y);
                        }
                    }
                    // the row's maximum over both halves of the tile
                    volatile float* t2 = tops + (tc & 1u) * 512;  // the partner may still read the last tile's
                    t2[wg * 128 + r] = top;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(kLBarTop + 4 * (int)g + quad));
                    ok = loss_wait(bar(kLBarTop + 4 * (int)g + quad), tc++ & 1u, wt, 113);
                    if (!ok) break;
                    top = fmaxf(top, t2[(wg ^ 1u) * 128 + r]);
                    const float m = fmaxf(off, top);
                    // nothing visible yet (every class masked): any finite offset gives 2^-inf = 0
                    const float m0 = m == -CUDART_INF_F ? 0.0f : m;
                    const float corr = off == -CUDART_INF_F ? 0.0f : ex2_approx(off - m0);
                    off = m;
                    if (with_o && half == 0 && ringed) ring[((rc + i) & 3u) * 128 + r] = m;
                    const float sub = F32 ? 14.0f - m0 : -m0;
                    const float2 sub2 = make_float2(sub, sub);
                    float2 ts = make_float2(0.f, 0.f);
#pragma unroll (F32 ? 1 : 4)
                    for (int q = 0; q < 4; ++q) {
                        uint32_t x[16];
                        tmem_ld32x32b_x16(t_s + 16u * q, x);
                        tmem_ld_wait16(x);
                        drop_named(x, q);
                        float2 pr[8];
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 e = SLOTS ? make_float4(0.f, 0.f, 0.f, 0.f) : lds128(tab + 4u * (16 * q + j));
                            float2 a = __ffma2_rn(as_pair(x[j], x[j + 1]), mul, make_float2(e.x, e.y));
                            float2 b = __ffma2_rn(as_pair(x[j + 2], x[j + 3]), mul, make_float2(e.z, e.w));
                            a = __fadd2_rn(a, sub2);
                            b = __fadd2_rn(b, sub2);
                            pr[j / 2] = make_float2(ex2_approx(a.x), ex2_approx(a.y));
                            pr[j / 2 + 1] = make_float2(ex2_approx(b.x), ex2_approx(b.y));
                            ts = __fadd2_rn(ts, __fadd2_rn(pr[j / 2], pr[j / 2 + 1]));
                        }
                        if (with_o) store_probs<F32, TWO>(t_s + 16u * q, pr);
                    }
                    const float t = F32 ? (ts.x + ts.y) * (1.0f / 16384.0f) : ts.x + ts.y;
                    sum = fmaf(sum, corr, t);
                } else {
                    const float2 le = make_float2(lane_e, lane_e);
                    // f32: 1 / gs, as gs is a power of two
                    const float gs_up = __uint_as_float(0x7f000000u - __float_as_uint(gs));
                    bool labelled = false;  // most tiles have none of a warp's classes
                    if (lw.next < lw.end) {
                        window_use(lw, ent, lane, (int)half);
                        labelled = lw.groups != 0u || lw.last < 8;
                    }
                    float2 ts = make_float2(0.f, 0.f);
#pragma unroll (F32 ? 1 : 4)
                    for (int q = 0; q < 4; ++q) {
                        uint32_t x[16];
                        tmem_ld32x32b_x16(t_s + 16u * q, x);
                        tmem_ld_wait16(x);
                        float2 pr[8];
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 e = lds128(tab + 4u * (16 * q + j));
                            float2 a = __ffma2_rn(as_pair(x[j], x[j + 1]), mul, make_float2(e.x, e.y));
                            float2 b = __ffma2_rn(as_pair(x[j + 2], x[j + 3]), mul, make_float2(e.z, e.w));
                            if (!SLOTS) {
                                a = __fadd2_rn(a, le);
                                b = __fadd2_rn(b, le);
                            }
                            pr[j / 2] = make_float2(ex2_approx(a.x), ex2_approx(a.y));
                            pr[j / 2 + 1] = make_float2(ex2_approx(b.x), ex2_approx(b.y));
                            if (F32 || gs != 0.0f) {  // f32: the factors; bf16: their signs, where one is negative
                                const float4 f = lds128(tab + 512u + 4u * (16 * q + j));
                                pr[j / 2] = __fmul2_rn(pr[j / 2], make_float2(f.x, f.y));
                                pr[j / 2 + 1] = __fmul2_rn(pr[j / 2 + 1], make_float2(f.z, f.w));
                            }
                        }
                        // the labels' gradients, 8 columns (rows of x) at a time through a patch of
                        // shared memory: entries scatter into it, each lane then takes its class's row
#pragma unroll
                        for (int h = 0; h < 2 && labelled; ++h) {
                            const int group = 2 * q + h;
                            bool any = false;
                            while (true) {
                                if ((lw.groups >> group) & 1u) {
                                    any = true;
                                    if (lw.group == group)
                                        *reinterpret_cast<volatile float*>(
                                            gbase + (patch - base) + 4u * (uint32_t)(lw.e.x & 31) * kPatchRow +
                                            4u * (uint32_t)((lw.e.x >> 5) & 7)) =
                                            F32 ? __int_as_float(lw.e.y) * gs_up : __int_as_float(lw.e.y);
                                }
                                if (group < lw.last) break;  // the window reaches beyond this group, or is the last
                                lw.e = lw.n;
                                window_use(lw, ent, lane, (int)half);
                            }
                            if (any) {
                                __syncwarp();
                                const uint32_t row = patch + 4u * (uint32_t)lane * kPatchRow;
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const uint4 d = lds128u(row + 16u * j);
                                    float2 &lo = pr[4 * h + 2 * j], &hi = pr[4 * h + 2 * j + 1];
                                    if (d.x != (uint32_t)kNoPatch) lo.x = __uint_as_float(d.x);
                                    if (d.y != (uint32_t)kNoPatch) lo.y = __uint_as_float(d.y);
                                    if (d.z != (uint32_t)kNoPatch) hi.x = __uint_as_float(d.z);
                                    if (d.w != (uint32_t)kNoPatch) hi.y = __uint_as_float(d.w);
                                    sts128u(row + 16u * j, make_uint4((uint32_t)kNoPatch, (uint32_t)kNoPatch,
                                                                      (uint32_t)kNoPatch, (uint32_t)kNoPatch));
                                }
                                __syncwarp();
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; j += 2) ts = __fadd2_rn(ts, __fadd2_rn(pr[j], pr[j + 1]));
                        store_probs<F32, TWO>(t_s + 16u * q, pr);
                    }
                    // bias gradient with the rounding error carried (up to thousands of tiles)
                    const float t = fmaf(ts.x + ts.y, F32 ? gs : 1.0f, carry);
                    const float nsum = sum + t;
                    carry = t - (nsum - sum);
                    sum = nsum;
                    lw.next = next_range.x;
                    lw.end = next_range.y;
                    ent += 256 * p.n_top;
                    lw.e = window_entry(lw, ent, lane);
                }
                if (!WPASS) nr = {next_named.x, next_named.y, next_named.w,
                                  named_entry(named_ent, next_named.x + lane, next_named.w)};
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kLBarPFull + 2 * (int)buf + (int)half));
                    mbar_arrive(bar(kLBarEmpty + (int)s));
                    if (!WPASS && with_o && half == 0 && ringed) mbar_arrive(bar(kLBarRing + (int)((rc + i) & 3u)));
                }
            }
            if (!ok) break;
            cc += n;
            if (ringed) rc += n;
            ok = loss_wait(bar(kLBarMsEmpty), (uc & 1u) ^ 1u, wt, 110);
            if (!ok) break;
            reinterpret_cast<float2*>(gbase + kMOffMs)[wg * 128 + r] =
                WPASS ? make_float2(sum, carry) : make_float2(off, sum);
            mbar_arrive(bar(kLBarMsFull));
        }
    } else {
        setmaxnreg_inc<kAddRegs>();
        // -------------------------------------------------------------- adding warpgroups
        // acc is relative to `off`, the largest offset of the tiles so far (row pass; the two softmax
        // warpgroups each keep their own running maximum).
        const uint32_t g = (uint32_t)(warp - 20) >> 2;
        const int quad = warp & 3, r = quad * 32 + lane;
        const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + kTO + 64u * g;
        const volatile float* ring = reinterpret_cast<const volatile float*>(gbase + kMOffRing);
        const int f0 = 64 * (int)g;
        uint32_t fc = 0, rc = 0, uc = 0;  // products taken, of them with an offset; units
        bool ok = true;
        for (int u; ok && (u = lunit_at((int)uc, p)) >= 0; ++uc) {
            const LUnit U = lunit(u, p);
            float off = -CUDART_INF_F;
            float2 acc[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i] = make_float2(0.f, 0.f);
            if (with_o) {
                const int every = add_every(U.own);
                for (int c = U.c0; c < U.c1; c += every, ++fc) {
                    float om = F32 ? chain_load(p.str_scale + c) : 1.0f;  // value of one unit of the product
                    if (F32) om *= WPASS ? chain_load(p.g_scale + c) : 1.0f / 16384.0f;
                    float corr = 1.0f;
                    if (!WPASS && every == 1) {
                        ok = loss_wait(bar(kLBarRing + (int)(rc & 3u)), (rc >> 2) & 1u, wt, 112);
                        if (!ok) break;
                        const float o = ring[(rc & 3u) * 128 + r];
                        const float m = fmaxf(off, o);
                        corr = off == m ? 1.0f : off == -CUDART_INF_F ? 0.0f : ex2_approx(off - m);
                        if (o != m) om *= ex2_approx(o - m);
                        off = m;
                        ++rc;
                    }
                    const bool grow = !WPASS && !__all_sync(0xffffffffu, corr == 1.0f);
                    ok = loss_wait(bar(kLBarOFull), fc & 1u, wt, 109);
                    if (!ok) break;
                    tc_fence_after();
                    const float2 om2 = make_float2(om, om), c2 = make_float2(corr, corr);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (f0 + 16 * q < feat) {
                            uint32_t v[16];
                            tmem_ld32x32b_x16(t_o + 16u * q, v);
                            tmem_ld_wait16(v);
                            if (grow) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) acc[8 * q + j] = __fmul2_rn(acc[8 * q + j], c2);
                            }
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                acc[8 * q + j] = __ffma2_rn(as_pair(v[2 * j], v[2 * j + 1]), om2, acc[8 * q + j]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(kLBarOEmpty));
                }
                if (!ok) break;
                const bool direct = WPASS && p.dw != nullptr;
                if (direct && U.own * 128 + r < p.n) {
                    // a thread's class row, 16 bytes at a time
                    const size_t at = (size_t)(U.own * 128 + r) * p.k + f0;
#pragma unroll
                    for (int q = 0; q < (F32 ? 16 : 8); ++q) {
                        if constexpr (F32) {
                            if (f0 + 4 * q < p.k)
                                *reinterpret_cast<float4*>(static_cast<float*>(p.dw) + at + 4 * q) =
                                    make_float4(acc[2 * q].x, acc[2 * q].y, acc[2 * q + 1].x, acc[2 * q + 1].y);
                        } else if (f0 + 8 * q < p.k) {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 h = __floats2bfloat162_rn(acc[4 * q + j].x, acc[4 * q + j].y);
                                w[j] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.dw) + at + 8 * q) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                float* po = p.part_o + ((size_t)u * feat + f0) * 128 + r;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (!direct && f0 + 16 * q < feat) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            po[(size_t)(16 * q + 2 * j) * 128] = acc[8 * q + j].x;
                            po[(size_t)(16 * q + 2 * j + 1) * 128] = acc[8 * q + j].y;
                        }
                    }
                }
            }
            if (g == 0) {
                ok = loss_wait(bar(kLBarMsFull), uc & 1u, wt, 111);
                if (!ok) break;
                const float2* ms = reinterpret_cast<const float2*>(gbase + kMOffMs);
                const float2 a0 = ms[r], a1 = ms[128 + r], b0 = ms[256 + r], b1 = ms[384 + r];
                mbar_arrive(bar(kLBarMsEmpty));
                float2 out;
                if (WPASS) {
                    out = make_float2(((a0.x + a1.x) + (b0.x + b1.x)) + ((a0.y + a1.y) + (b0.y + b1.y)), 0.0f);
                } else {  // the halves of one parity share their offset
                    const float m = fmaxf(a0.x, b0.x);
                    const float k0 = a0.x == -CUDART_INF_F ? 0.0f : ex2_approx(a0.x - m);
                    const float k1 = b0.x == -CUDART_INF_F ? 0.0f : ex2_approx(b0.x - m);
                    out = make_float2(m, (a0.y + a1.y) * k0 + (b0.y + b1.y) * k1);
                }
                if (!WPASS || p.dw == nullptr)
                    p.part_ms[(size_t)u * 128 + r] = out;
                else if (p.db && U.own * 128 + r < p.n)
                    p.db[U.own * 128 + r] = out.x;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------- row kernel
namespace {

// A row's K slots over a group of 8 lanes: 16 per lane, in runs of kRun (one 16-byte load in the
// element type E): lane s of the group holds slots kRun (s + 8 j) + i, j < 16 / kRun, i < kRun.
template <int kRun>
__device__ __forceinline__ int lane_slot(int s, int i) {
    return kRun * (s + 8 * (i / kRun)) + i % kRun;
}

// A lane's 16 values of row `c` of a row-major [.][k] matrix (zero past k), as loaded: several rows'
// loads are in flight before the first is used.
template <bool F32>
struct WeightRow {
    static constexpr int kRun = F32 ? 4 : 8;
    uint4 u[16 / kRun];
    __device__ __forceinline__ void fetch(const void* w, long long c, int k, int s, bool vec) {
        using T = typename Elem<F32>::type;
        const T* a = static_cast<const T*>(w) + c * k;
#pragma unroll
        for (int j = 0; j < 16 / kRun; ++j) {
            const int k0 = kRun * (s + 8 * j);
            u[j] = make_uint4(0u, 0u, 0u, 0u);
            if (vec) {
                if (k0 < k) u[j] = __ldg(reinterpret_cast<const uint4*>(a + k0));
            } else {
                uint32_t x[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int i = 0; i < kRun; ++i) {
                    if (k0 + i >= k) continue;
                    if constexpr (F32)
                        x[i] = __float_as_uint(a[k0 + i]);
                    else
                        x[i / 2] |= (uint32_t)__bfloat16_as_ushort(a[k0 + i]) << (16 * (i % 2));
                }
                u[j] = make_uint4(x[0], x[1], x[2], x[3]);
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 16 / kRun; ++j) u[j] = make_uint4(0u, 0u, 0u, 0u);
    }
    // values 2 i and 2 i + 1
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (F32) {
            const uint4 q = u[i / 2];
            return i % 2 == 0 ? make_float2(__uint_as_float(q.x), __uint_as_float(q.y))
                              : make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
        } else {
            const uint4 q = u[i / 4];
            const uint32_t x = i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w;
            return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
        }
    }
};
template <int kRun>
__device__ __forceinline__ void shared_row(const float* row, int k, int s, float2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int k0 = lane_slot<kRun>(s, 2 * i);
        v[i] = make_float2(k0 < k ? row[k0] : 0.0f, k0 + 1 < k ? row[k0 + 1] : 0.0f);
    }
}
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// R rows of the features into shared memory (row stride k + 1), and back: coalesced along the
// layout's contiguous direction, every load of a thread in flight at once (k <= 128).
template <int R, int NT, class T>
struct RowLoad {
    static constexpr int kPer = R * 128 / NT;  // loads a thread
    float v[kPer];
    __device__ __forceinline__ void fetch(const T* x, long long row0, long long rows, int k, long long t_len) {
        if (t_len > 0) {
            const int r = threadIdx.x % R;
            const bool live = row0 + r < rows;
            const T* at = x + (live ? x_base(row0 + r, k, t_len) : 0);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int kk = threadIdx.x / R + i * (NT / R);
                v[i] = live && kk < k ? to_f32(at[kk * t_len]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {  // a warp's rows, a quarter each; or (R = 8) half a row a warp
                const int q = (threadIdx.x >> 5) * kPer + i, r = q / 4, kk = (threadIdx.x & 31) + 32 * (q % 4);
                v[i] = row0 + r < rows && kk < k ? to_f32(x[(row0 + r) * k + kk]) : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void put(int k, long long t_len, float* xs) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = (threadIdx.x >> 5) * kPer + i;
            const int r = t_len > 0 ? threadIdx.x % R : q / 4;
            const int kk = t_len > 0 ? threadIdx.x / R + i * (NT / R) : (threadIdx.x & 31) + 32 * (q % 4);
            if (kk < k) xs[r * (k + 1) + kk] = v[i];
        }
    }
};
template <int R, int NT, class T>
__device__ __forceinline__ void store_rows(T* x, long long row0, long long rows, int k, long long t_len,
                                           const float* xs) {
    if (t_len > 0) {
        const int r = threadIdx.x % R;
        if (row0 + r >= rows) return;
        T* at = x + x_base(row0 + r, k, t_len);
#pragma unroll 4
        for (int kk = threadIdx.x / R; kk < k; kk += NT / R) at[kk * t_len] = (T)xs[r * (k + 1) + kk];
    } else {
#pragma unroll
        for (int r = threadIdx.x >> 5; r < R; r += NT / 32) {
            if (row0 + r >= rows) return;
#pragma unroll 4
            for (int kk = threadIdx.x & 31; kk < k; kk += 32) x[(row0 + r) * k + kk] = (T)xs[r * (k + 1) + kk];
        }
    }
}

// A row's labels in a group of 8 lanes: their shares q into shared memory as (class or -1, q), and
// sum_i q_i log q_i; a share may round to zero. False when the row has none (it is then ignored), or
// none is asked for.
__device__ __forceinline__ bool group_labels(const LossLabels& L, long long row, bool live, int s, int2* ent,
                                             float& entropy) {
    entropy = 0.0f;
    if (L.target) {
        const int t = live ? L.target[row] : -1;
        const bool valid = is_class(t, L.n);
        if (s == 0) ent[0] = make_int2(valid ? t : -1, __float_as_int(1.0f));
        __syncwarp();
        return valid;
    }
    const long long at = row * L.n_top;
    float top = -CUDART_INF_F;
    bool any = false;
    for (int e = s; e < L.n_top; e += 8) {
        int c = live ? L.top_idx[at + e] : -1;
        c = is_class(c, L.n) ? c : -1;
        const float u = c >= 0 ? L.top_logits[at + e] * L.inv_temp : -CUDART_INF_F;
        if (u == -CUDART_INF_F) c = -1;  // of no share: as absent
        ent[e] = make_int2(c, __float_as_int(u));
        any |= c >= 0;
        top = fmaxf(top, u);
    }
    top = group_max(top);
    const bool valid = group_max(any ? 1.0f : 0.0f) > 0.0f;
    float sum = 0.0f;
    for (int e = s; e < L.n_top; e += 8)
        if (ent[e].x >= 0) sum += expf(__int_as_float(ent[e].y) - top);
    sum = group_sum(sum);
    const float log_sum = logf(sum);
    float h = 0.0f;
    for (int e = s; e < L.n_top; e += 8) {
        if (ent[e].x < 0) continue;
        const float u = __int_as_float(ent[e].y) - top, q = expf(u) / sum;
        // (a share that rounds to zero holds the row to nothing)
        if (q != 0.0f) h = fmaf(q, u - log_sum, h);
        ent[e] = make_int2(ent[e].x, __float_as_int(q));
    }
    entropy = group_sum(h);
    __syncwarp();
    return valid;
}

// Rows l0 .. l0 + R - 1 of the units u0 .. u0 + ns - 1's partial tiles [feat][128], weighted and
// added in the units' order, into os [R][feat + 1]. A thread owns one row and every
// (NT / R)-th feature, and keeps all of its features' loads of a unit in flight: with few rows the
// work is split over many units, and their latency is what this join costs.
template <int R, int NT, bool WEIGHTED>
__device__ __forceinline__ void join_units(const float* part_o, size_t u0, int ns, int feat, int l0, const float* wgt,
                                           float* os) {
    constexpr int kStep = NT / R, kPer = 128 / kStep;
    const int r = threadIdx.x % R, f0 = threadIdx.x / R;
    float a[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) a[i] = 0.0f;
    const float* po = part_o + u0 * feat * 128 + (size_t)f0 * 128 + l0 + r;
#pragma unroll(R == 8 ? 8 : 4)
    for (int s = 0; s < ns; ++s, po += (size_t)feat * 128) {
        const float w = WEIGHTED ? wgt[s * R + r] : 1.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (f0 + i * kStep < feat) a[i] = fmaf(chain_load(po + (size_t)i * kStep * 128), w, a[i]);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (f0 + i * kStep < feat) os[r * (feat + 1) + f0 + i * kStep] = a[i];
}

}  // namespace

// One block per R rows (32; 8 where that leaves most SMs idle, and then of 512 threads where there are
// fewer blocks than SMs: each joins many units). Joins the class ranges of a row block (the largest
// offset, the sums and weighted rows brought to it: U and O over the classes that the row does not
// name); then 8 lanes per row: the labels' logits z_i as f32 products, e_i = 2^(z_i - M), S = U + sum_i
// e_i, lse = M + log S, the labels' gradients f (e_i / S - q_i), the loss, and
// dx = f (O / S + sum_i (e_i / S - q_i) W_ci).
// Where one label holds the row, e / S - q is the difference of two numbers near 1. It is taken, for
// the entry with the largest share, as (e_t (1 - q_t) - q_t (S - e_t)) / S with both differences summed
// from the other entries; a single entry (q = 1) so has -U / S, and its loss log(1 + U / e), to f32's
// precision of themselves.
template <bool F32, int R, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 3 : 1) loss_rows_kernel(const __grid_constant__ LossRowParams p) {
    using T = typename Elem<F32>::type;
    extern __shared__ __align__(16) float sm[];
    float* xs = sm;                                           // [R][k + 1]
    float* os = xs + R * (p.k + 1);                           // [R][feat + 1]
    float* wgt = os + R * (p.feat + 1);                       // [n_splits][R]
    int2* ents = reinterpret_cast<int2*>(wgt + R * p.n_splits);  // [R][n_top] (R is even: 8-byte aligned)
    float* zs = reinterpret_cast<float*>(ents + R * p.lab.n_top);  // [R][n_top]: z_i, then e_i / S - q_i
    int* places = reinterpret_cast<int*>(zs + R * p.lab.n_top);    // [R][n_top]: sp_pos
    constexpr int kG = NT / R;                 // threads that share a row's ranges
    constexpr int kRun = F32 ? 4 : 8;
    __shared__ float red[kG][R];
    __shared__ float s_off[R], s_sum[R];
    __shared__ float s_top[R], s_factor[R];
    __shared__ bool s_last;
    const int tid = threadIdx.x;
    launch_next();
    wait_previous();
    const long long row0 = (long long)blockIdx.x * R;
    const int mb = (int)(row0 >> 7), l0 = (int)(row0 & 127);
    const int ns = mb < p.whole_units ? 1 : p.n_splits;
    const size_t u0 = mb < p.whole_units ? (size_t)mb
                                         : (size_t)p.whole_units + (size_t)(mb - p.whole_units) * p.n_splits;

    RowLoad<R, NT, T> xv;
    xv.fetch(static_cast<const T*>(p.x), row0, p.rows, p.k, p.t_len);
    const int jr = tid % R, jg = tid / R;
    if (ns == 1) {
        // one unit has the whole class range: nothing to join
        const float2 ms = chain_load(p.part_ms + u0 * 128 + l0 + jr);
        if (jg == 0) {
            s_off[jr] = ms.x;
            s_sum[jr] = ms.y;
        }
        if (p.dx) {
            constexpr int kPer = 128 / kG;
            const float* po = p.part_o + u0 * p.feat * 128 + l0 + jr;
            float a[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                a[i] = jg + i * kG < p.feat ? chain_load(po + (size_t)(jg + i * kG) * 128) : 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (jg + i * kG < p.feat) os[jr * (p.feat + 1) + jg + i * kG] = a[i];
        }
    } else {
        float m = -CUDART_INF_F;
        for (int s = jg; s < ns; s += kG) {
            const float o = chain_load(p.part_ms + (u0 + s) * 128 + l0 + jr).x;
            wgt[s * R + jr] = o;
            m = fmaxf(m, o);
        }
        red[jg][jr] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kG; ++i) m = fmaxf(m, red[i][jr]);
        const float m0 = m == -CUDART_INF_F ? 0.0f : m;
        float sum = 0.0f;
        __syncthreads();
        for (int s = jg; s < ns; s += kG) {
            const float k = ex2_approx(wgt[s * R + jr] - m0);
            wgt[s * R + jr] = k;
            sum = fmaf(chain_load(p.part_ms + (u0 + s) * 128 + l0 + jr).y, k, sum);
        }
        red[jg][jr] = sum;
        __syncthreads();
        if (jg == 0) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kG; ++i) sum += red[i][jr];
            s_off[jr] = m;
            s_sum[jr] = sum;
        }
        __syncthreads();
        if (p.dx) join_units<R, NT, true>(p.part_o, u0, ns, p.feat, l0, wgt, os);
    }
    xv.put(p.k, p.t_len, xs);
    __syncthreads();
    if (tid < 8 * R) {  // (R = 8: two warps have rows)
        const bool vec = p.k % kRun == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15u) == 0;
        const int r = tid >> 3, s = tid & 7;
        const long long row = row0 + r;
        const bool live = row < p.rows;
        int2* ent = ents + r * p.lab.n_top;
        float* zr = zs + r * p.lab.n_top;
        int* place = places + r * p.lab.n_top;
        for (int e = s; live && e < p.lab.n_top; e += 8) place[e] = chain_load(p.sp_pos + row * p.lab.n_top + e);
        float entropy;
        const bool valid = group_labels(p.lab, row, live, s, ent, entropy);
        const float f = live ? p.lab.temp * (p.row_grad ? p.row_grad[row] : 1.0f) : 0.0f;
        float* xr = xs + r * (p.k + 1);
        float2 x[8];
        shared_row<kRun>(xr, p.k, s, x);

        // the labels' logits in log2 units over T, rounded as the scores are
        constexpr int kBatch = 2;
        for (int e0 = 0; e0 < p.lab.n_top; e0 += kBatch) {
            int c[kBatch];
            float b[kBatch], z[kBatch];
            WeightRow<F32> w[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                c[j] = valid && e0 + j < p.lab.n_top ? ent[e0 + j].x : -1;
                b[j] = 0.0f;
                if (c[j] >= 0) {
                    w[j].fetch(p.w, c[j], p.k, s, vec);
                    if (p.bias) b[j] = __ldg(p.bias + c[j]);
                } else {
                    w[j].clear();
                }
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                float2 z2 = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 8; ++i) z2 = __ffma2_rn(x[i], w[j].pair(i), z2);
                z[j] = z2.x + z2.y;
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) z[j] += __shfl_xor_sync(0xffffffffu, z[j], o);
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (s == 0 && e0 + j < p.lab.n_top)
                    zr[e0 + j] = p.slots ? (z[j] + b[j]) * p.logit_scale
                                         : fmaf(z[j], p.logit_scale, b[j] * p.logit_scale);
        }
        __syncwarp();

        // the row's sum, from the classes that it does not name (U, relative to off) and its labels.
        // A class named again keeps its first entry, with both shares.
        float kl2 = 0.0f, q_top = -1.0f, z_max = -CUDART_INF_F;
        int top = p.lab.n_top, count = 0;
        for (int e = s; e < p.lab.n_top; e += 8) {
            if (!valid || ent[e].x < 0) continue;
            ++count;
            z_max = fmaxf(z_max, zr[e]);
        }
        count = __reduce_add_sync(0xffu << (tid & 24), count);
        z_max = group_max(z_max);
        const float off = s_off[r];
        const float m = fmaxf(off, z_max), m0 = m == -CUDART_INF_F ? 0.0f : m;
        const float scale_u = off == -CUDART_INF_F ? 0.0f : ex2_approx(off - m0);
        const float u_sum = s_sum[r] * scale_u;
        bool again = false;
        for (int e = s; e < p.lab.n_top; e += 8) {
            if (!valid || ent[e].x < 0) continue;
            if (place[e] < 0) again = true;
        }
        if (__any_sync(0xffffffffu, again)) {
            for (int e = s; e < p.lab.n_top; e += 8) {
                const int2 en = ent[e];
                if (!valid || en.x < 0 || place[e] < 0) continue;
                float q = __int_as_float(en.y);
                for (int j = 0; j < p.lab.n_top; ++j)  // (only entries that stay are written, only others read)
                    if (j != e && ent[j].x == en.x) q += __int_as_float(ent[j].y);
                ent[e].y = __float_as_int(q);
            }
            __syncwarp();
            for (int e = s; e < p.lab.n_top; e += 8)
                if (valid && ent[e].x >= 0 && place[e] < 0) ent[e].x = -1;
            __syncwarp();
        }
        for (int e = s; e < p.lab.n_top; e += 8) {
            if (!valid || ent[e].x < 0) continue;
            const float q = __int_as_float(ent[e].y);
            if (q > q_top) {
                q_top = q;
                top = e;
            }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            const float oq = __shfl_xor_sync(0xffffffffu, q_top, o);
            const int ot = __shfl_xor_sync(0xffffffffu, top, o);
            if (oq > q_top || (oq == q_top && ot < top)) {
                q_top = oq;
                top = ot;
            }
        }
        float e_rest = 0.0f, q_rest = 0.0f;
        for (int e = s; e < p.lab.n_top; e += 8) {
            if (!valid || ent[e].x < 0 || e == top) continue;
            e_rest += ex2_approx(zr[e] - m0);
            q_rest += __int_as_float(ent[e].y);
        }
        e_rest = group_sum(e_rest);
        q_rest = group_sum(q_rest);
        const float z_top = top < p.lab.n_top ? zr[top] : -CUDART_INF_F;
        const float e_top = ex2_approx(z_top - m0), others = u_sum + e_rest, total = others + e_top;
        const float inv = 1.0f / total, lse2 = m + log2f(total);
        __syncwarp();
        // the labels' gradients over f, and their part of the loss
        float largest = u_sum * inv;
        int2* tile_ent = p.sp_ent + (row >> 7) * 128 * p.lab.n_top;
        for (int e = s; e < p.lab.n_top; e += 8) {
            if (!valid || ent[e].x < 0) continue;
            const float q = __int_as_float(ent[e].y), z = zr[e];
            if (q != 0.0f) kl2 = fmaf(q, z - lse2, kl2);
            const float d = e == top ? (e_top * q_rest - q * others) * inv : fmaf(ex2_approx(z - m0), inv, -q);
            zr[e] = d;
            largest = fmaxf(largest, fabsf(d));
            tile_ent[place[e]].y = __float_as_int(f * d);
        }
        kl2 = group_sum(kl2);
        largest = group_max(largest);
        __syncwarp();
        if (F32 && s == 0) {
            s_top[r] = valid ? fabsf(f) * largest : 0.0f;
            s_factor[r] = valid ? fabsf(f) : 0.0f;
        }
        if (s == 0) {
            float e = -CUDART_INF_F;  // no share of anything
            if (valid) e = F32 ? -lse2 : log2f(fabsf(f)) - lse2;
            p.row_tab[(size_t)(row >> 7) * 256 + (row & 127)] = e;
        }
        if (live && s == 0) {
            float loss = entropy - kl2 * kLn2;
            if (count == 1 && q_top == 1.0f && z_top < CUDART_INF_F)  // one label: what the other classes leave
                loss = z_top >= off ? log1pf(s_sum[r] * ex2_approx(off - z_top))
                                    : (off - z_top) * kLn2 + logf(s_sum[r] + ex2_approx(z_top - off));
            if (p.loss) p.loss[row] = valid ? loss * p.lab.temp * p.lab.temp : 0.0f;
            if (p.lse) p.lse[row] = valid ? lse2 * kLn2 : 0.0f;
        }
        if (p.dx) {
            float2 d[8];
            shared_row<kRun>(os + r * (p.feat + 1), p.k, s, d);
            const float2 ku = make_float2(scale_u * inv, scale_u * inv);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = __fmul2_rn(d[i], ku);
            for (int e0 = 0; e0 < p.lab.n_top; e0 += kBatch) {
                WeightRow<F32> w[kBatch];
                float2 g[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int c = valid && e0 + j < p.lab.n_top ? ent[e0 + j].x : -1;
                    g[j] = make_float2(0.f, 0.f);
                    if (c >= 0) {
                        w[j].fetch(p.w, c, p.k, s, vec);
                        g[j].x = g[j].y = zr[e0 + j];
                    } else {
                        w[j].clear();
                    }
                }
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[i] = __ffma2_rn(g[j], w[j].pair(i), d[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k0 = lane_slot<kRun>(s, 2 * i);
                if (k0 < p.k) xr[k0] = valid ? f * d[i].x : 0.0f;
                if (k0 + 1 < p.k) xr[k0 + 1] = valid ? f * d[i].y : 0.0f;
            }
        }
    }
    if (F32 || p.dx) __syncthreads();
    if (p.dx) store_rows<R, NT>(static_cast<T*>(p.dx), row0, p.rows, p.k, p.t_len, xs);
    if constexpr (F32) {
        // The scale of a tile's gradients: its largest comes to 2^13, so that the weight pass's fp16 pairs
        // hold down to 2^-38 of it (of the largest factor f alone, the gradients that confident rows leave
        // would be below the pairs' last step). The last of a tile's blocks knows it.
        if (tid < 32) {
            const float t = warp_max(tid < R ? s_top[tid] : 0.0f), g = warp_max(tid < R ? s_factor[tid] : 0.0f);
            if (tid == 0) {
                p.tile_top[(size_t)mb * kLossTopSlots + l0 / R] = make_float2(t, g);
                __threadfence();
                s_last = atomicAdd(p.tile_done + mb, 1) == kLossTile / R - 1;
            }
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (tid >= kLossTile) return;
        float t = 0.0f, g = 0.0f;
#pragma unroll
        for (int i = 0; i < kLossTile / R; ++i) {
            const float2 v = chain_load(p.tile_top + (size_t)mb * kLossTopSlots + i);
            t = fmaxf(t, v.x);
            g = fmaxf(g, v.y);
        }
        // (times the features' scale it must stay a normal number, and the factors themselves finite)
        const int sh = min(min(shift_to(t, 13), 96), shift_to(g, 100));
        float* factor = p.row_tab + (size_t)mb * 256 + 128 + tid;
        *factor = chain_load(factor) * pow2i(sh);
        if (tid == 0) p.g_scale[mb] = pow2i(-sh);
    }
}

// One block per R classes (32, or 8 as above): the row ranges' partial sums added in their order,
// transposed through shared memory into dW [n][k].
template <bool F32, int R>
__global__ void __launch_bounds__(256) loss_reduce_kernel(const __grid_constant__ LossReduceParams p) {
    using T = typename Elem<F32>::type;
    extern __shared__ float sm[];  // [R][feat + 1]
    wait_previous();
    const int j0 = (int)blockIdx.x * R, tile = j0 >> 7, l0 = j0 & 127;
    const int ns = tile < p.whole_units ? 1 : p.n_splits;
    const size_t u0 = tile < p.whole_units ? (size_t)tile
                                           : (size_t)p.whole_units + (size_t)(tile - p.whole_units) * p.n_splits;
    join_units<R, 256, false>(p.part_o, u0, ns, p.feat, l0, nullptr, sm);
    if (p.db && threadIdx.x < R && j0 + (int)threadIdx.x < p.n) {
        float a = 0.0f;
        for (int s = 0; s < ns; ++s) a += chain_load(p.part_ms + (u0 + s) * 128 + l0 + threadIdx.x).x;
        p.db[j0 + threadIdx.x] = a;
    }
    __syncthreads();
    T* dw = static_cast<T*>(p.dw);
#pragma unroll
    for (int r = threadIdx.x >> 5; r < R; r += 8) {
        if (j0 + r < p.n) {
            for (int kk = threadIdx.x & 31; kk < p.k; kk += 32)
                dw[(long long)(j0 + r) * p.k + kk] = (T)sm[r * (p.feat + 1) + kk];
        }
    }
}

// ---------------------------------------------------------------------------- packed heads
// Class table at temperature T: scale / T and bias / T (the decode kernel then decodes z / T).
__global__ void __launch_bounds__(256) loss_table_kernel(const float* __restrict__ ctab, long long n, float inv_temp,
                                                         float* __restrict__ out) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = ctab[i] * inv_temp;
}

namespace {

// A lane's 16 K slots of a packed weight's class c, in units of its class-table scale: runs of 8
// (fp16 images), or 16 in a row (compact).
template <int FORM>
__device__ __forceinline__ void packed_row(const uint8_t* tiles, int c, int s, float2 (&v)[8]) {
    const int tile = c >> 7, r = c & 127;
    if constexpr (FORM == 1) {
        const uint8_t* a = tiles + (size_t)tile * kTile8Bytes + image8_offset(r, 16 * s);
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(a));
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w = x[i / 2] >> (16 * (i % 2));
            v[i] = make_float2((float)(int)(w & 255u) - 128.0f, (float)(int)((w >> 8) & 255u) - 128.0f);
        }
    } else {
        const uint8_t* a = tiles + (size_t)tile * (FORM == 2 ? 2 * kTileBytes : kTileBytes);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t off = image_chunk(r, s + 8 * j);
#pragma unroll
            for (int part = 0; part < (FORM == 2 ? 2 : 1); ++part) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(a + part * kTileBytes + off));
                const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
                    v[4 * j + i] = part ? __fadd2_rn(v[4 * j + i], f) : f;
                }
            }
        }
    }
}

}  // namespace

// One block per 32 rows, 8 lanes per row: the logits of the row's labels and of its argmax as f32
// products with the packed weight. lse = z[argmax] / T + log(sum of exponentials relative to it); a loss
// is formed from differences of logits.
// Rows whose class range was split are joined here, from the decode kernel's partial (maximum, sum,
// argmax) rows.
template <int FORM>
__global__ void __launch_bounds__(256) loss_score_kernel(const __grid_constant__ LossScoreParams p) {
    extern __shared__ __align__(16) float xs[];  // [32][k + 1], then [32][n_top] int2
    constexpr int kRun = FORM == 1 ? 16 : 8;
    int2* ents = reinterpret_cast<int2*>(xs + kLossRows * (p.k + 1));
    const long long row0 = (long long)blockIdx.x * kLossRows;
    const int r = threadIdx.x >> 3, s = threadIdx.x & 7;
    const long long row = row0 + r;
    const bool live = row < p.rows;
    RowLoad<kLossRows, 256, float> xv;
    xv.fetch(p.x, row0, p.rows, p.k, p.t_len);
    // The caller's features and labels are there already; only what the decode kernel writes is waited for.
    // (That kernel has no trigger, so this one starts as its last blocks end: the reads above run beside
    // their end and the flush after it, no earlier.)
    int2* ent = ents + r * p.lab.n_top;
    float entropy;
    const bool valid = group_labels(p.lab, row, live, s, ent, entropy);
    xv.put(p.k, p.t_len, xs);
    wait_previous();
    int best = 0;
    float sum = 1.0f, m = CUDART_NAN_F;  // m: the decode kernel's maximum, where it is known
    if (row >= p.split_row0 && live) {
        m = -CUDART_INF_F;
        sum = 0.0f;
        best = 0x7fffffff;
        // eight ranges' entries in flight at a time: their latency is what this join costs
        const float4* part = p.partial + (size_t)(row - p.split_row0);
        const size_t step = (size_t)(p.rows - p.split_row0);
        for (int i0 = s; i0 < p.n_splits; i0 += 64) {
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = i0 + 8 * j < p.n_splits ? chain_load(part + (size_t)(i0 + 8 * j) * step)
                                               : make_float4(-CUDART_INF_F, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = __float_as_int(v[j].z);
                if (v[j].x > m) {
                    sum = (m == -CUDART_INF_F ? 0.0f : sum * ex2_approx(m - v[j].x)) + v[j].y;
                    m = v[j].x;
                    best = c;
                } else if (v[j].x != -CUDART_INF_F) {
                    sum += v[j].y * ex2_approx(v[j].x - m);
                    if (v[j].x == m) best = min(best, c);
                } else if (isnan(v[j].y)) {
                    sum = CUDART_NAN_F;
                }
            }
        }
        // lanes of a group that had no range, or only masked classes, bring nothing
        const uint32_t group = 0xffu << (threadIdx.x & 24);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(group, m, o), os = __shfl_xor_sync(group, sum, o);
            const int ob = __shfl_xor_sync(group, best, o);
            const float M = fmaxf(m, om);
            if (M != -CUDART_INF_F) {
                sum = (m == -CUDART_INF_F ? 0.0f : sum * ex2_approx(m - M)) +
                      (om == -CUDART_INF_F ? 0.0f : os * ex2_approx(om - M));
                best = m == om ? min(best, ob) : m > om ? best : ob;
            } else {
                sum += os;
            }
            m = M;
        }
    } else if (live) {
        best = chain_load(p.idx + row);
        sum = 1.0f / chain_load(p.prob + row);
    }
    best = min(max(best, 0), p.lab.n - 1);
    __syncthreads();
    if (live) {
        const int* cls = p.lab.target ? p.lab.target + row : p.lab.top_idx + row * p.lab.n_top;
        bool bad = false;
        for (int e = s; e < p.lab.n_top; e += 8) bad |= cls[e] >= p.lab.n;
        if (bad) atomicOr(p.status + kStatusBadClass, 1);
    }
    float2 x[8];
    shared_row<kRun>(xs + r * (p.k + 1), p.k, s, x);
    auto logit = [&](int c) -> float {
        float2 w[8], z = make_float2(0.f, 0.f);
        packed_row<FORM>(p.tiles, c, s, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) z = __ffma2_rn(x[i], w[i], z);
        const float* t = p.ctab + (size_t)(c >> 7) * kCtabFloats + (c & 127);
        return fmaf(group_sum(z.x + z.y), __ldg(t), __ldg(t + kBlockN)) * p.lab.inv_temp;
    };
    // lse - z[best] from the other classes' sum. That is relative to the tensor core's z[best], a sum that
    // rounds toward zero and is some 2^-22 of itself short; where the row's maximum is at hand the sum is
    // brought to the f32 logit (z in log2 units in two parts, so that the difference keeps its digits).
    const float z_best = logit(best);
    float rest = sum < 1.0f ? 0.0f : sum - 1.0f;
    const float z_hi = z_best * 1.4426950408889634f;
    const float z_lo = fmaf(z_best, 1.4426950408889634f, -z_hi);
    const float off = (m - z_hi) - z_lo;
    if (fabsf(off) < 1.0f) rest *= ex2_approx(off);
    const float gap = log1pf(rest), lse = z_best + gap;
    float zq = 0.0f;
#pragma unroll 2
    for (int e = 0; e < p.lab.n_top; ++e) {
        const int2 c = ent[e];
        const bool here = valid && c.x >= 0 && __int_as_float(c.y) != 0.0f;
        const float z = logit(here ? c.x : 0);
        if (here) zq = fmaf(__int_as_float(c.y), (z - z_best) - gap, zq);
    }
    if (live && s == 0) {
        if (p.loss) p.loss[row] = valid ? (entropy - zq) * p.lab.temp * p.lab.temp : 0.0f;
        if (p.lse) p.lse[row] = valid ? lse : 0.0f;
    }
}

// ------------------------------------------------------------------------------- launchers
namespace {
// (counts, starts, entries; the norms' four partial sums)
constexpr int pack_smem_bytes(int w_tiles, int n_top) {
    return 4 * w_tiles * (2 * kPackWarps + 4) + 128 * n_top * 4;
}
constexpr int kPackSmemMax = pack_smem_bytes(kLossMaxClasses / 128, kLossMaxTop) + 2048;
static_assert(kPackSmemMax <= 226 * 1024, "shared memory per block");
int rows_smem_bytes(int r, int k, int feat, int n_splits, int n_top) {
    return r * ((k + 1 + feat + 1 + n_splits) * 4 + n_top * 16);
}
constexpr int kRowsSmemMax = 32 * ((2 * 129 + kLossMaxSplits) * 4 + kLossMaxTop * 16);
int score_smem_bytes(int k, int n_top) { return kLossRows * ((k + 1) * 4 + n_top * 8); }
// Blocks of 32 rows would leave SMs idle: four times as many of 8.
bool few_blocks(int tiles, int sms) { return tiles * (kLossTile / 32) < 2 * sms; }
template <class K>
cudaError_t smem_attr(K* k, int bytes) {
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
}  // namespace

cudaError_t loss_kernel_setup(int* wrong_registers) {
    cudaError_t e;
    void (*const main_kernels[])(LossMainParams) = {
        loss_main_kernel<true, false, false>,        loss_main_kernel<true, true, false>,
        loss_main_kernel<false, false, false>,       loss_main_kernel<false, true, false>,
        loss_main_kernel<false, false, true>,        loss_main_kernel<false, true, true>,
        loss_main_kernel<false, false, false, true>, loss_main_kernel<false, true, false, true>,
        loss_main_kernel<false, false, true, true>,  loss_main_kernel<false, true, true, true>};
    *wrong_registers = 0;
    for (auto k : main_kernels) {
        cudaFuncAttributes a{};
        if ((e = cudaFuncGetAttributes(&a, k)) != cudaSuccess) return e;
        if (!split_fits(a.numRegs)) *wrong_registers = a.numRegs;
        if ((e = smem_attr(k, kMSmemBytes)) != cudaSuccess) return e;
    }
    if ((e = smem_attr(loss_pack_kernel<true>, kPackSmemMax)) != cudaSuccess) return e;
    if ((e = smem_attr(loss_pack_kernel<false>, kPackSmemMax)) != cudaSuccess) return e;
    if ((e = smem_attr(loss_rows_kernel<true, 32, 256>, kRowsSmemMax)) != cudaSuccess) return e;
    return smem_attr(loss_rows_kernel<false, 32, 256>, kRowsSmemMax);
}

namespace {
// A launch that may start before the kernel ahead of it in the stream has ended (that kernel says
// when; wait_previous() then waits for its end).
template <class P>
cudaError_t launch_chained(void (*kernel)(P), int grid, int threads, int smem, cudaStream_t stream, const P& p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}
}  // namespace

cudaError_t launch_loss_pack(const LossPackParams& p, bool f32, cudaStream_t stream) {
    const int grid = p.w_tiles + p.x_tiles;
    const int labels = pack_smem_bytes(p.w_tiles, p.lab.n_top);
    LossPackParams q = p;
    q.norm_smem = (labels + 3) / 4;
    const int smem = 4 * q.norm_smem + (p.slots && p.t_len > 0 ? 2048 : 0);
    if (f32)
        loss_pack_kernel<true><<<grid, kPackThreads, smem, stream>>>(q);
    else
        loss_pack_kernel<false><<<grid, kPackThreads, smem, stream>>>(q);
    return cudaGetLastError();
}

cudaError_t launch_loss_main(const LossMainParams& p, bool f32, bool slots, bool weight_pass, int grid,
                             cudaStream_t stream) {
    void (*k)(LossMainParams);
    if (f32)
        k = weight_pass ? loss_main_kernel<true, true, false> : loss_main_kernel<true, false, false>;
    else if (p.str_tiles <= kTwoPartTiles && weight_pass)
        k = slots ? loss_main_kernel<false, true, true, true> : loss_main_kernel<false, true, false, true>;
    else if (p.str_tiles <= kTwoPartTiles)
        k = slots ? loss_main_kernel<false, false, true, true> : loss_main_kernel<false, false, false, true>;
    else if (slots)
        k = weight_pass ? loss_main_kernel<false, true, true> : loss_main_kernel<false, false, true>;
    else
        k = weight_pass ? loss_main_kernel<false, true, false> : loss_main_kernel<false, false, false>;
    return launch_chained(k, grid, kMainThreads, kMSmemBytes, stream, p);
}

cudaError_t launch_loss_rows(const LossRowParams& p, bool f32, int sms, cudaStream_t stream) {
    const int tiles = (int)((p.rows + kLossTile - 1) / kLossTile);  // the last tile's padding rows too
    const int r = few_blocks(tiles, sms) ? 8 : 32;
    void (*k)(LossRowParams);
    const int grid = tiles * (kLossTile / r), threads = r == 8 && grid <= sms ? 512 : 256;
    if (r == 32)
        k = f32 ? loss_rows_kernel<true, 32, 256> : loss_rows_kernel<false, 32, 256>;
    else if (threads == 256)
        k = f32 ? loss_rows_kernel<true, 8, 256> : loss_rows_kernel<false, 8, 256>;
    else
        k = f32 ? loss_rows_kernel<true, 8, 512> : loss_rows_kernel<false, 8, 512>;
    return launch_chained(k, grid, threads, rows_smem_bytes(r, p.k, p.feat, p.n_splits, p.lab.n_top), stream, p);
}

cudaError_t launch_loss_reduce(const LossReduceParams& p, bool f32, int sms, cudaStream_t stream) {
    const int r = few_blocks((p.n + kLossTile - 1) / kLossTile, sms) ? 8 : 32;
    void (*k)(LossReduceParams);
    if (f32)
        k = r == 32 ? loss_reduce_kernel<true, 32> : loss_reduce_kernel<true, 8>;
    else
        k = r == 32 ? loss_reduce_kernel<false, 32> : loss_reduce_kernel<false, 8>;
    return launch_chained(k, (p.n + r - 1) / r, 256, r * (p.feat + 1) * 4, stream, p);
}

cudaError_t launch_loss_table(const float* ctab, long long n_floats, float inv_temp, float* out, cudaStream_t stream) {
    loss_table_kernel<<<(int)((n_floats + 255) / 256), 256, 0, stream>>>(ctab, n_floats, inv_temp, out);
    return cudaGetLastError();
}

cudaError_t launch_loss_score(const LossScoreParams& p, cudaStream_t stream) {
    const int grid = (int)((p.rows + kLossRows - 1) / kLossRows);
    void (*k)(LossScoreParams) = p.form == 0   ? loss_score_kernel<0>
                                 : p.form == 1 ? loss_score_kernel<1>
                                               : loss_score_kernel<2>;
    return launch_chained(k, grid, 256, score_smem_bytes(p.k, p.lab.n_top), stream, p);
}

}  // namespace rh
