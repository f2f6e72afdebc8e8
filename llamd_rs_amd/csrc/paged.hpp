// paged.hpp -- arguments of the paged-cache kernels (paged_store.hip, paged_attend.hpp) and their launchers. The entry
// points (paged.cpp) check everything that the host can see; the kernels check what lies on the device (sequence starts,
// lengths, page ids) before it becomes an address.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace llamd {

enum PagedType { PT_F32 = 0, PT_F16 = 1, PT_BF16 = 30 };  // ggml's numbers
constexpr int SCALE_BLOCK = 16, SCALE_LOG = 4;            // positions of 8-bit pages that share a scale

// The cache and the batch (llamd_hip_pages or llamd_hip_pages8, llamd_hip_batch), as the kernels take them.
struct PagedArgs {
    void *k, *v;           // [n_page][n_kv_head][page][hd], [n_page][n_kv_head][hd][page]
    const int32_t *start;  // [n_seq + 1]; null: sequence s has token s
    const int32_t *len;    // [n_seq]
    const int32_t *table;  // [n_seq][max_page]
    int n_page, page_log, n_kv_head, hd;
    int n_seq, n_tok, max_page;
    int n_head, group;  // group = n_head / n_kv_head
    uint8_t *k_scale, *v_scale;  // 8-bit pages: [n_page][n_kv_head][page / 16]
};

struct PagedStoreArgs {
    PagedArgs p;
    const float *x[3];        // Q (may be null), K, V
    int ld[3];                // floats between tokens' rows
    const float *norm[2];     // of Q and K heads, each may be null
    float eps;
    const double *freqs;      // [n_rot / 2] radians per position
    int n_rot, interleaved;
    float mscale;
    void *q_out;
};

struct PagedAttendArgs {
    PagedArgs p;
    const void *q;
    void *out;
    int out_f32;
    float scale;              // times log2(e): the kernels' exponentials are powers of two
    const int32_t *group_at;  // decode: [n_groups + 1] first sequence of each group; null: no groups
    const int32_t *shared;    // decode: [n_groups] positions that a group shares
    int n_groups;
};

// paged_store.hip
int launch_paged_store(const PagedStoreArgs &a, int type, hipStream_t st);
// paged_attend_*.hip: a prompt batch or a decode batch
int launch_paged_attend_f32(const PagedAttendArgs &a, bool decode, hipStream_t st);
int launch_paged_attend_f16(const PagedAttendArgs &a, bool decode, hipStream_t st);
int launch_paged_attend_bf16(const PagedAttendArgs &a, bool decode, hipStream_t st);
int launch_paged_attend_e4m3(const PagedAttendArgs &a, bool decode, hipStream_t st);
// paged8_store.hip
int launch_paged8_store(const PagedStoreArgs &a, hipStream_t st);

}  // namespace llamd
