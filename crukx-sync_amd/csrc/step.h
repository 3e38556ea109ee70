// The training step's kernels (step.hip): argument layouts and launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace crx {

enum : int { kBf16 = 0, kF16 = 1, kF32 = 2 };
enum : int { kMeanToken = 0, kMeanSequence = 1, kSum = 2 };

// One value per position (b, t), at any strides.
template <typename T>
struct At {
    const T *p;
    int64_t sb, st;
};

// Logits and what says which of them count: rows of `vocab` elements, row b * tokens + t at
// x + b * sb + t * st.
struct RowsIn {
    const void *x;
    int64_t sb, st;
    uint32_t seqs, tokens, vocab;
    uint32_t rows, row0;  // all rows; the launch's first
    const void *ids;
    int64_t ids_sb, ids_st;
    int32_t id_bytes;
    At<uint8_t> mask;  // p null: no position is masked
    float c;           // log2(e) / temperature
    float inv_temp, inv_temp_lo;  // 1 / temperature, and what it was rounded by
};

struct ScoreOut {
    float *logp;
    float *entropy;  // or null
    float2 *stats;   // or null: the row's largest logit and the sum of its exponentials
};

struct PolicyIn {
    At<float> old, adv, ref;  // ref.p null: no KL term
    float low, high;          // the ratio's limits, 1 - clip_low and 1 + clip_high
    float kl, scale;
    int32_t reduction;
    const uint32_t *counts;  // [seqs] unmasked positions, then their sum and the number of sequences that
                             // have any; null: no position is masked
};

struct PolicyOut {
    float *logp;
    float2 *stats;  // or null
    float *slope;   // or null
    float *terms;   // [3][rows] weighted loss, KL and clipped of every row
    void *grad;     // or null
};

// The gradient of a row: a (1[j = y] - p_j) - h p_j (ln p_j + H), with a and h given per position.
struct GradIn {
    const float2 *stats;
    const float *slope;    // a, contiguous, or null:
    At<float> up_logp;     //   a = up_logp / temperature (p null: 0)
    At<float> up_entropy;  // h = up_entropy / temperature (p null: 0)
    const float *entropy;  // H (with up_entropy)
    const float *upstream; // a factor of every row, in device memory, or null
    int32_t unless_one;    // nothing to do where it is 1
    void *grad;
};

// Rows that are too few to give every CU one are cut into parts of `size` elements (a multiple of 8), n of them a
// row (1: rows are not cut), each on a workgroup of its own.
struct Parts {
    float *stat;  // [rows][n][3] the parts' statistics
    uint32_t n, size;
    uint32_t *counts;  // where one workgroup more counts the mask, or null
};
constexpr uint32_t kPartRows = 256;  // rows from which they are not cut: one for each of the chip's CUs (512: 300 rows of
                                     // 152064 took 55 us cut and 54 whole, of 20011 17 and 13)
constexpr uint32_t kMostParts = 64;  // a wavefront joins a row's parts
constexpr uint32_t kPartLeast = 2048;
constexpr int kPartBlock = 256;
Parts parts_of(uint64_t rows, uint64_t vocab);
// elements of a row that a workgroup of the gradient's pass takes (4000 rows of 152064 bf16: 425 us, of 4096 434, of
// 16384 460, of 32768 481)
constexpr uint64_t kGradPart = 8192;
constexpr uint32_t kIdleBlocks = 2048;  // workgroups of that pass where it is likely to have nothing to do
constexpr uint32_t kFewPositions = 65536, kFewSeqs = 4096;  // whose mask one workgroup counts

void launch_mask_counts(const RowsIn &x, uint32_t *counts, hipStream_t s);
void launch_score(const RowsIn &x, const Parts &p, const ScoreOut &o, int dtype, hipStream_t s);
void launch_policy(const RowsIn &x, const Parts &parts, const PolicyIn &p, const PolicyOut &o, int dtype, hipStream_t s);
void launch_policy_sums(const float *terms, uint32_t rows, float scale, float *loss, float *kl, float *clipped,
                        hipStream_t s);
void launch_rows_grad(const RowsIn &x, const GradIn &g, int dtype, hipStream_t s);

// Lists of tensors of one type go to the kernels as arguments (no upload): so many in one launch, under the
// 4 KiB that a launch's arguments take.
constexpr uint32_t kNormTensors = 192, kAdamTensors = 72;
constexpr uint32_t kUnit = 1024;        // elements that lists are dealt out to workgroups by
constexpr uint32_t kNormBlocks = 2048;  // workgroups of the norm's pass, most: 8 on each of 256 CUs
constexpr uint32_t kNormShare = 8, kClipShare = 4, kAdamShare = 2;  // units of a workgroup's share
// Units of a launch, most.  The passes that write go over long lists in several launches: in one, the workgroups on
// different parts of the chip drift apart, and reads and writes that far apart cost bandwidth.  AdamW of 1.5e9 weights
// (with its norm), us: 7840 in one launch, 7660 in launches of 2^18 units, 7580 of 2^17, 7580 of 2^16, 7630 of 2^15, 7790 of
// 2^14; of 41e6 weights 201 in launches of 2^16 and more, 209 of 2^15, 223 of 2^14.  The norm only reads: 2200 for 7.6e9
// gradients in one launch, 2470 in launches of 2^18.
constexpr uint32_t kNormUnits = 1u << 30, kClipUnits = 1u << 18, kAdamUnits = 1u << 16;
// Workgroups of a launch of the clip, which take several shares where there are more: usually there is nothing to clip,
// and then they are what the launch costs.  7.6e9 bf16 gradients, us with nothing to clip and to clip them: 139 and 4870;
// with a workgroup for each share 441 and 4840; in launches of 2^19 units 73 and 5140; in one launch of a workgroup for
// each share of 16 units 100 and 5560.
constexpr uint32_t kClipBlocks = 16384;
constexpr uint64_t kKeepBytes = 192ULL << 20;  // gradients that the 256 MB last-level cache keeps for the next pass

struct NormList {
    void *p[kNormTensors];
    uint64_t n[kNormTensors];
    uint32_t first[kNormTensors + 1];  // units before the tensor's
    uint32_t count;                    // tensors
};

struct AdamList {
    void *w[kAdamTensors];
    float *master[kAdamTensors], *m[kAdamTensors], *v[kAdamTensors];
    const void *g[kAdamTensors];
    uint64_t n[kAdamTensors];
    uint32_t first[kAdamTensors + 1];
    uint32_t count;
};

struct AdamArgs {
    double keep;      // 1 - lr * weight_decay
    float beta1, beta2, one_less_beta1, one_less_beta2;
    float rate;       // lr / (1 - beta1^step)
    float root;       // 1 / sqrt(1 - beta2^step)
    float eps;
    const float *norm;  // or null
    float max_norm;
};

static_assert(sizeof(NormList) + 64 <= 4096 && sizeof(AdamList) + sizeof(AdamArgs) <= 4096, "a launch's arguments");

// partial[b], for every workgroup b of `blocks`: its squares' sum, added to what is there where b < used.
// keep: the caches should hold the gradients, which the next pass reads (launch_clip: as they were kept)
void launch_norm_part(const NormList &l, int dtype, double *partial, uint32_t used, bool keep, uint32_t blocks, hipStream_t s);
void launch_norm_sum(const double *partial, uint32_t n, float *norm, hipStream_t s);
void launch_clip(const NormList &l, int dtype, const float *norm, float max_norm, bool keep, uint32_t shares, hipStream_t s);
void launch_adamw(const AdamList &l, int wtype, int gtype, const AdamArgs &a, uint32_t blocks, hipStream_t s);

void timing_begin(const char *name, hipStream_t s);
void timing_end(const char *name, hipStream_t s);

}  // namespace crx
