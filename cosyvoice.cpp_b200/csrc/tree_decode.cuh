// tree_decode.cuh -- attention of a tree of drafted tokens over a typed KV cache.
//
// For sequence s with L committed positions and n drafted nodes, row r = (node i,
// query head g of the KV head's group of G) attends the keys 0 .. L - 1 of the
// cache and the drafted keys its mask row lists:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c q.k_j - m),  c = scale log2 e,
// in one pass with a running maximum m and sum per row.  The keys of a sequence
// form ceil(L / T) cache tiles and ceil(n / T) draft tiles of T keys; a split is a
// run of consecutive tiles, and splits leave (m, sum) and an unnormalized output
// per row for tree_combine_kernel.
#pragma once

#include "common.cuh"
#include "launch.cuh"
#include "internal.h"

namespace cvattn {
namespace tree {

constexpr int kD = 64;      // head size

struct Args {
    const float* q;
    int64_t q_nb_node, q_nb_seq;
    float* out;
    int64_t out_nb_node, out_nb_seq;
    float* lse;
    const uint8_t *k, *v, *kd, *vd;
    int64_t k_nb1, k_nb2, v_nb1, v_nb2, kd_nb1, kd_nb2, vd_nb1, vd_nb2;
    const uint64_t *k_seq_ptrs, *v_seq_ptrs;
    const int32_t *kv_len, *n_nodes;
    const uint32_t* mask;
    int64_t mask_nb_seq;
    int mask_words;
    int k_type, v_type;
    int n_seq, max_nodes, Hq, Hkv, G, max_kv_len;
    int tile;                    // keys per tile
    int split_tiles, n_splits;   // tiles per split, most splits of a sequence
    float scale_log2;
    float* ws_ml;                // [seq][KV head][split][max_nodes * G][2]
    float* ws_o;                 // [seq][KV head][split][max_nodes * G][64]
    int* status;
};

// The lengths of one sequence; (0, 0) if they, or its rows' addresses, are out of range.
struct Lens {
    int L, n, tiles, cache_tiles;
};
__device__ __forceinline__ Lens lens_of(const Args& a, int s, bool record) {
    Lens x;
    x.L = a.kv_len[s];
    x.n = a.n_nodes ? a.n_nodes[s] : a.max_nodes;
    bool bad = x.L < 0 || x.L > a.max_kv_len || x.n < 0 || x.n > a.max_nodes;
    if (a.k_seq_ptrs && (a.k_seq_ptrs[s] & (a.k_type == kF32 ? 3 : 1))) bad = true;
    if (a.v_seq_ptrs && (a.v_seq_ptrs[s] & (a.v_type == kF32 ? 3 : 1))) bad = true;
    if (bad) {
        if (record) record_status(a.status, kStatusBadLength);
        x.L = x.n = 0;
    }
    x.cache_tiles = (x.L + a.tile - 1) / a.tile;
    x.tiles = x.n == 0 ? 0 : x.cache_tiles + (a.kd ? (x.n + a.tile - 1) / a.tile : 0);
    return x;
}

__device__ __forceinline__ const uint8_t* seq_base(const uint64_t* ptrs, const uint8_t* base, int64_t nb2, int s) {
    return ptrs ? reinterpret_cast<const uint8_t*>(ptrs[s]) : base + (int64_t)s * nb2;
}

__device__ __forceinline__ bool node_sees(const Args& a, int s, int i, int j) {
    if (!a.mask) return j <= i;
    return (a.mask[(int64_t)s * a.mask_nb_seq + (int64_t)i * a.mask_words + (j >> 5)] >> (j & 31)) & 1u;
}

}  // namespace tree
}  // namespace cvattn
