// Launch parameters of the training-loss kernels (loss_kernels.cu), shared with the host
// dispatch (rechead_abi.cu). Plain C types only.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace rh {

constexpr int kLossTile = 128;            // rows (classes) per operand tile
constexpr int kLossImage = 128 * 128 * 2;  // one 16-bit tile image: 128 rows x 128 K slots
constexpr int kLossMaxTop = 64;           // teacher entries per row
constexpr int kLossMaxClasses = 1 << 17;  // labels are counted by 32 classes in shared memory (4,096 bins)
constexpr int kLossRows = 32;             // rows per block of the score kernel
constexpr int kLossTopSlots = 16;         // blocks of the row kernel per tile at most
constexpr int kLossMaxSplits = 148;       // ranges that an own tile's work is split into at most
// Device status word (status[2], non-zero: set): a target or teacher class at or above the class count;
// the row or entry was taken as absent. Apart from status[0] and [1], which every host call on the slot
// reads: a bad label is its own call's, told by the next rh_sync.
constexpr int kStatusBadClass = 2;
constexpr int kStatusWords = 3;

// What a row is held to: a target class, or a teacher's top logits. Exactly one of target and
// top_idx is set.
struct LossLabels {
    const int32_t* target;     // [rows], negative: the row is ignored
    const int32_t* top_idx;    // [rows][n_top], negative: the entry is absent
    const float* top_logits;   // [rows][n_top]
    int n_top;                 // 1 with target
    int n;                     // classes
    float temp;                // T
    float inv_temp;            // 1 / T
};

// Operand tiles of a training step: features and weight as tensor-core images, the class table,
// the rows' gradient factors and the labels sorted by class tile.
struct LossPackParams {
    const void* x;             // [rows][k], or [rows / t_len][k][t_len] (t_len > 0)
    const void* w;             // [n][k]
    const float* bias;         // [n] or null
    const float* row_grad;     // [rows] d total / d loss_r, or null: 1
    LossLabels lab;
    long long rows, t_len;
    int k, x_tiles, w_tiles;
    float logit_scale;         // log2(e) / T
    uint8_t* x_img;            // x_tiles images (f32: high image, then low image)
    uint8_t* w_img;
    float* x_scale;            // [x_tiles] value of one unit of the image (f32; a power of two)
    float* w_scale;            // [w_tiles]
    float* class_e;            // [w_tiles][128] bias * log2(e) / T; padding classes -inf
    float* row_tab;            // [x_tiles][256]. f32: 128 x (-lse, log2 units; written by the row kernel),
                               // 128 x gradient factor, scaled by the row kernel to g_scale's unit. bf16: 128 x
                               // (log2 |factor| - lse; by the row kernel), 128 x the factor's sign
    float* g_scale;            // [x_tiles] f32: value of one unit of the tile's gradients (a power of two; by
                               // the row kernel); bf16: 1 where a factor is negative, else 0
    int* tile_done;            // [x_tiles] f32: blocks of the row kernel that are done, set to 0
    int slots;                 // bf16, k <= 125: K slots k..k+2 hold the bias in three parts (weight) and 1
                               // (features), so that the scores come with their bias
    float* x_norm;             // slots: [x_tiles][128] |x_r|
    float2* w_bound;           // slots: [w_tiles] (largest |w_j|, largest bias in log2 units)
    int norm_smem;             // set by the launcher: first float of the norms' shared memory
    int2* sp_off;              // [x_tiles][4 w_tiles] label ranges (first, end) by 32 classes
    int2* sp_ent;              // [x_tiles][128 n_top]: (row << 5 | class within its 32, bits of the gradient
                               // dz; by the row kernel)
    int* sp_pos;               // [x_tiles][128 n_top]: an entry's place in its tile's sp_ent; -1: absent, or
                               // of a class that an earlier entry of the row names
    int* status;
};

// One pass over (own tile, streamed tiles): see loss_main_kernel.
struct LossMainParams {
    const uint8_t* own;        // images of the stationary operand
    const uint8_t* str;        // images of the streamed operand
    const float* own_scale;    // per tile (f32)
    const float* str_scale;
    const float* col_tab;      // per streamed tile: class_e (128 floats) or row_tab (256 floats)
    const float* lane_e;       // weight pass: class_e of the own classes (not with slots)
    const float* x_norm;       // row pass, slots
    const float2* w_bound;
    const float* g_scale;      // weight pass: per streamed tile
    const int2* sp_off;
    const int2* sp_ent;
    int n_top;
    int own_tiles, str_tiles;
    int ksteps;                // K steps of 16
    int whole_units, n_splits, tiles_per_split;
    float logit_scale;
    float* part_o;             // [units][16 ksteps][128], or null: only (offset, sum) (row pass)
    float2* part_ms;           // [units][128]: row pass (offset, sum); weight pass (bias gradient, 0)
    // Weight pass of one unit per own tile: dW [n][k] and db [n] (or null) straight from the unit,
    // instead of part_o / part_ms. 16-byte rows and pointer.
    void* dw;
    float* db;
    int n, k;
    int* status;
    unsigned long long timeout_ns;
};

// Rows of a training step after the row pass: loss, lse, the feature gradient, the row table and the
// labels' own gradients.
struct LossRowParams {
    const void* x;
    const void* w;
    const float* bias;
    const float* row_grad;
    LossLabels lab;
    long long rows, t_len;
    int k, feat;
    int whole_units, n_splits;
    float logit_scale;
    int slots;                 // bias within the scores (bf16), or added to them in log2 units
    const float* part_o;
    const float2* part_ms;
    const int* sp_pos;
    int2* sp_ent;
    float2* tile_top;          // [x_tiles][kLossTopSlots] f32: a block's largest |dz| and |factor|
    int* tile_done;
    float* g_scale;
    float* row_tab;
    float* loss;               // [rows] or null
    float* lse;                // [rows] or null
    void* dx;                  // as x, or null
};

struct LossReduceParams {      // weight and bias gradient from the units' partial tiles
    const float* part_o;
    const float2* part_ms;
    int n, k, feat;
    int whole_units, n_splits;
    void* dw;                  // [n][k]
    float* db;                 // [n] or null
};

// Scores of a packed head: (idx, prob) of the decode kernel at temperature T -> loss, lse.
struct LossScoreParams {
    const float* x;
    long long rows, t_len;
    int k;
    LossLabels lab;
    const uint8_t* tiles;      // packed weight
    const float* ctab;         // class table (scale, bias), at T = 1
    int form;                  // 0 fp16 image of int8, 1 compact int8, 2 FP32 (hi, lo)
    const int32_t* idx;        // rows below split_row0
    const float* prob;
    const float4* partial;     // rows from split_row0 on: [n_splits][rows - split_row0], as HeadParams::partial
    long long split_row0;
    int n_splits;
    float* loss;
    float* lse;
    int* status;
};

// wrong_registers: 0, or the registers a thread of a main kernel whose register split would not be met
// (it is then not to be launched).
cudaError_t loss_kernel_setup(int* wrong_registers);
cudaError_t launch_loss_pack(const LossPackParams& p, bool f32, cudaStream_t stream);
cudaError_t launch_loss_main(const LossMainParams& p, bool f32, bool slots, bool weight_pass, int grid,
                             cudaStream_t stream);
cudaError_t launch_loss_rows(const LossRowParams& p, bool f32, int sms, cudaStream_t stream);
cudaError_t launch_loss_reduce(const LossReduceParams& p, bool f32, int sms, cudaStream_t stream);
cudaError_t launch_loss_table(const float* ctab, long long n_floats, float inv_temp, float* out, cudaStream_t stream);
cudaError_t launch_loss_score(const LossScoreParams& p, cudaStream_t stream);

}  // namespace rh
