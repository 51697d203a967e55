// kv.h — the paged KV cache as its kernels see it (kv_cache.hip writes and
// reads rows, kv_attention.hip attends over them, decode.hip serves from it).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/welvet_hip.h"

namespace wv {

// One layer's pools. Positions are held in blocks of 32 keys of one page and
// KV head, block index kv_block() below, each in the order that the matrix
// instructions of the attention read it:
//   k  16-byte units [unit u][key 32]: the codes of dims u*16/E .. of one key
//      (E bytes per code)
//   v  groups [octet o 4][dim][8 codes]: the 8 keys of an octet for one dim
//   s  floats [octet o 4][2][8]: the K scales, then the V scales of an octet
// Octet o = 2a + b of a block holds the keys 16a + 8(j/4) + 4b + j%4, j = 0..7:
// the keys whose scores one lane ends with after a 32x32 score product
// (kv_octet_key). Codes are always finite (int8 codes biased by 128), a row
// that held a NaN or an infinity has a NaN scale: reading any block is safe,
// and a masked key needs only its scale and probability dropped.
struct KvView {
    uint8_t* k;
    uint8_t* v;
    float* s;
    int n_kv, hd, type;
    int page_shift;  // log2 page_size, 5..8
    int n_pages;
};

constexpr int kKvBlock = 32;      // keys of a block
constexpr int kKvScales = 64;     // floats of a block's scales
inline __host__ __device__ int64_t kv_block(const KvView& c, int64_t page, int head, int offset) {
    return ((page * c.n_kv + head) << (c.page_shift - 5)) + (offset >> 5);
}
inline __host__ __device__ int kv_octet_key(int o, int j) {
    return 16 * (o >> 1) + 8 * (j >> 2) + 4 * (o & 1) + (j & 3);
}
// Octet and index in it of key kk (0..31).
inline __host__ __device__ void kv_key_octet(int kk, int& o, int& j) {
    o = 2 * (kk >> 4) + ((kk >> 2) & 1);
    j = 4 * ((kk >> 3) & 1) + (kk & 3);
}
inline int kv_code_bytes(int type) { return type == WV_KV_F16 ? 2 : 1; }

struct KvCache {
    wv_kv_config c{};
    int device = 0;
    uint8_t* base = nullptr;
    size_t bytes = 0;
    size_t layer_bytes = 0, code_bytes = 0;  // per layer: k codes, v codes, scales
    KvView layer(int l) const {
        uint8_t* p = base + size_t(l) * layer_bytes;
        int sh = 0;
        while ((1 << sh) < c.page_size) ++sh;
        return KvView{p, p + code_bytes, reinterpret_cast<float*>(p + 2 * code_bytes), c.n_kv_heads, c.head_dim,
                      c.type, sh, c.n_pages};
    }
};

// Copies the description of cache `h`; false if the handle is unknown.
bool kv_lookup(uint64_t h, KvCache& out);

int launch_kv_write(const KvView& c, const float* k, const float* v, int64_t ks, int64_t vs, const int64_t* slots,
                    int n, hipStream_t s);
int launch_kv_read(const KvView& c, const int64_t* slots, int n, float* k, float* v, int64_t ks, int64_t vs,
                   hipStream_t s);

// An attention call: the batch, its rows, and how it is cut. `splits` ranges
// of the keys (1: none); with more, part holds n_tokens * n_heads * splits
// partial rows of hd + 4 floats.
struct KvAttn {
    KvView c;
    const float* q;
    float* out;
    float* part;
    const int32_t *cu, *kv_len, *pages;
    int64_t qs, os;
    int n_seqs, n_tokens, max_pages;
    int n_heads, window;
    int splits;
    bool many;  // long sequences by the kernel of 128-row tiles
    bool once;  // one block reads a sequence's keys of a KV head
    float scale;
    // Sequences in groups that share their first keys: of the splits the first `lead` are ranges of a group's shared
    // keys, which all of its rows take from its first sequence's pages, the others ranges of a sequence's own.
    const int32_t *group_cu, *group_shared;
    int n_groups, lead;
};
// Which kernels a call takes and into how many key ranges it is cut (max_pages: as many as sequences hold), and
// the floats of its partials.
struct KvPlan {
    bool many, once;
    int splits;
    double us;  // about what it takes
};
KvPlan kv_attn_plan(const KvView& c, int n_seqs, int n_tokens, int max_pages, int max_q, int n_heads, int window);
size_t kv_attn_part_floats(const KvView& c, int n_tokens, int n_heads, int splits);
int launch_kv_attn(const KvAttn& a, hipStream_t s);
// With groups: whether that is faster than `whole`, attention over whole sequences, and into how many ranges the shared
// and the own keys are cut.
struct KvGroupPlan {
    bool use;
    int lead, own;
};
KvGroupPlan kv_attn_group_plan(const KvView& c, int n_seqs, int n_tokens, int max_pages, int n_heads, int window,
                               int n_groups, int max_shared, const KvPlan& whole);
int launch_kv_attn_groups(const KvAttn& a, const KvGroupPlan& p, hipStream_t s);

}  // namespace wv
