// C-ABI entry points of the attention over the 4-bit cache (kernels:
// attn_mx4_impl.h, instantiated per activation type in attn_mx4_{bf16,f16}.hip).
#include <algorithm>

#include "attn_mx4_impl.h"
#include "attn_ws.h"

using namespace fxpr;
using namespace fxpr::attn;
using namespace fxpr::attn::m4;

namespace {

constexpr int64_t kMaxGridZ = 65535;
// records above which a launch runs unsplit
constexpr int64_t kMx4WsMax = int64_t(1) << 30;

struct Planned {
  Mx4Plan p;
  WsLayout ws;
};

// Split policy (bf16, 32 query heads over 8 kv heads of size 128, the cache as
// empty_cache lays it out; a chunk is 512 keys).
// 16-row workgroups split when there are chunks to hand out and the launch is
// small, or its lengths may differ and it is not large (a split leaves a record
// per chunk): up to 128 workgroups from two chunks on (16 requests of 1000 keys
// 11.7 us, unsplit 12.4; 24 of them 14.1 against 12.7), up to 1024 from four (64
// requests of 1000 .. 8000 keys 70 us, unsplit 104; all of 8000 121 against 114;
// 128 of 500 .. 4000 76 against 84, all of 4000 125 against 113), none beyond
// (256 requests of 1000 .. 8000 keys 278 us, unsplit 261; all of 8000 493 against
// 398). About 6144 workgroups, eight rounds of the card, even the lengths out,
// and 12 splits where that is fewer (64 requests of 2000 .. 16000 keys: 12 splits
// 145 us, 4 160, 32 145; 128 of 1000 .. 8000 12 splits 138, 8 144); beyond 128 a
// request alone gains nothing (64000 keys 24.3 us, 64 splits 24.9; over one kv
// head 13.7 against 18.1). A window evens the lengths by itself: up to 384
// workgroups (the last where equal lengths gain: 48 requests of 4000 keys 51 us,
// unsplit 58; 83 requests under a window of 1024, f16, head size 64: 26.2 us,
// unsplit 24.0).
// The prompts' workgroups take two row sets (128 rows) where a launch has two for
// every CU, or so many chunks that splits make it about one; smaller launches
// end sooner with one (512 new tokens alone 23.5 us, with two 32; 128 over 2048
// keys 30 against 38, over 4096 39 against 41, over 8192 64 against 56; 2 x 512
// over 2048 93 against 106, 512 over 2048 69 against 62).
// They split while fewer than two fall to a CU, and up to that: 512 new tokens
// over 4096 keys 94 us with 4 splits, 205 unsplit, 97 with 8; 128 over 16000 97 us
// with 16, 788 unsplit; 4 x 256 over 4096 180 us with 2, 209 unsplit; with 512
// workgroups, 2048 over 4096, 249 us unsplit, 292 with 2. Of two or three chunks
// only up to 128 workgroups (128 over 1000 keys 29 us, unsplit 40; 8 x 64 over
// 1000 46 against 41).
Planned plan_mx4(int num_requests, int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int page_size,
                 int max_query_len, int max_blocks, int window, int int_bits, int requested) {
  Planned r;
  const int group = num_heads / num_kv_heads;
  const int64_t slots = std::max<int64_t>(chunk_slots(max_blocks, page_size), 1);
  const int64_t max_rows = int64_t(max_query_len > 1 ? max_query_len : 1) * group;
  r.p.prompt = max_rows >= kPrefillRows;
  const int64_t qtiles = std::min<int64_t>(cdiv(max_rows, QROWS), r.p.prompt ? kShortTiles : int64_t(1) << 40);
  const int64_t wgs16 = int64_t(num_requests) * num_kv_heads * qtiles;
  // chunks that a row's keys can touch
  const int64_t chunks = window > 0 ? std::min(slots, cdiv(int64_t(window) + max_query_len, TILE * CT) + 1) : slots;
  auto prompt_wgs = [&](int sets) { return std::max<int64_t>(cdiv(num_tokens * num_heads, int64_t(sets) * PQROWS), 1); };
  r.p.sets = row_sets(int_bits, head_dim);
  const int64_t wgs2 = prompt_wgs(2);
  if (wgs2 < 512 && (chunks < 4 || wgs2 * chunks < 256 || (chunks == 4 && wgs2 >= 256))) r.p.sets = 1;
  const int64_t wgsp = prompt_wgs(r.p.sets);
  int64_t s16 = 1, sp = 1;
  if (requested >= 1) {
    s16 = sp = std::min<int64_t>({int64_t(requested), slots, kMaxGridZ});
  } else {
    // (the tokens that the shortest request has when all others have the most: no
    // split, so no combine launch, for a request of a few rows that is not there)
    const bool only_long =
        r.p.prompt && (num_tokens - int64_t(num_requests - 1) * max_query_len) * group >= kPrefillRows;
    if (wgs16 <= (chunks < 4 ? 128 : window > 0 ? 384 : 1024) && !only_long)
      s16 = std::min(chunks, std::clamp<int64_t>(6144 / wgs16, 12, 128));
    if (r.p.prompt && wgsp < (chunks < 4 ? 129 : 512)) sp = std::min(cdiv(512, wgsp), chunks);
  }
  auto layout = [&](int64_t rows) { return ws_layout(rows, num_heads, head_dim, int_bits, true, slots); };
  if (sp > 1 || (s16 > 1 && !r.p.prompt)) {
    r.ws = layout(num_tokens);
    if (r.ws.total > kMx4WsMax) {
      r.ws = WsLayout{};
      if (!r.p.prompt || requested >= 1) s16 = 1;
      sp = 1;
    }
  }
  if (r.ws.total == 0 && s16 > 1) {
    // only the short requests leave records: room for their tokens alone
    const int64_t cap = std::min<int64_t>(max_query_len, std::max<int64_t>((kPrefillRows - 1) / group, 1));
    r.p.tok_cap = int(cap);
    r.ws = layout(int64_t(num_requests) * cap);
    if (r.ws.total > kMx4WsMax) {
      r.ws = WsLayout{};
      r.p.tok_cap = 0;
      s16 = 1;
    }
  }
  r.p.splits = int(s16);
  r.p.pq_splits = int(sp);
  return r;
}

bool page_ok(int page_size) { return page_size >= 16 && (page_size & (page_size - 1)) == 0; }
bool dim_ok(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

}  // namespace

extern "C" int64_t fxpr_attention_mx4_plan(int num_requests, int64_t num_tokens, int num_heads, int num_kv_heads,
                                           int head_dim, int page_size, int max_query_len, int max_blocks_per_seq,
                                           int window_size, int int_bits, int num_kv_splits, int32_t* plan) {
  if (plan) std::fill(plan, plan + 4, 0);
  if (num_requests <= 0 || num_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || !dim_ok(head_dim) ||
      max_blocks_per_seq <= 0 || !page_ok(page_size) || num_heads % num_kv_heads != 0 || num_kv_splits < 0 ||
      !valid_int_bits(int_bits))
    return 0;
  const Planned p = plan_mx4(num_requests, num_tokens, num_heads, num_kv_heads, head_dim, page_size, max_query_len,
                             max_blocks_per_seq, std::max(window_size, 0), int_bits, num_kv_splits);
  if (plan) {
    plan[0] = p.p.prompt ? 1 : 0;
    plan[1] = p.p.pq_splits;
    plan[2] = p.p.splits;
    plan[3] = p.p.tok_cap;
  }
  return p.ws.total;
}

extern "C" int fxpr_unified_attention_mx4(
    const void* q, const void* codes, const void* scales, void* o, int io_dtype, const int32_t* query_start_loc,
    const int32_t* seq_lens, const int32_t* block_table, const float* alibi_slopes, int num_requests,
    int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int page_size, int max_query_len,
    int max_blocks_per_seq, int64_t num_blocks, int64_t stride_q_token, int64_t stride_q_head,
    int64_t stride_codes_block, int64_t stride_codes_half, int64_t stride_codes_slot, int64_t stride_codes_head,
    int64_t stride_scales_block, int64_t stride_scales_half, int64_t stride_scales_slot, int64_t stride_scales_head,
    int64_t stride_o_token, int64_t stride_o_head, int64_t stride_bt_row, int is_causal, float softmax_scale_log2,
    float softcap_log2, int window_size, int int_bits, int frac_bits, int num_kv_splits, void* workspace,
    int64_t workspace_bytes, void* stream) {
  if (!valid_int_bits(int_bits) || frac_bits < 0 || frac_bits > 63) return FXPR_E_BITS;
  if (io_dtype != FXPR_DTYPE_BF16 && io_dtype != FXPR_DTYPE_F16) return FXPR_E_DTYPE;
  if (num_requests < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || !dim_ok(head_dim) ||
      !page_ok(page_size) || num_kv_splits < 0 || num_heads % num_kv_heads != 0)
    return FXPR_E_SHAPE;
  if (num_requests == 0 || num_tokens == 0) return FXPR_OK;
  if (max_blocks_per_seq <= 0 || num_blocks <= 0 || num_tokens > 0x7fffffff) return FXPR_E_SHAPE;
  if (!q || !codes || !scales || !o || !query_start_loc || !seq_lens || !block_table) return FXPR_E_ARG;
  // 16-byte loads of q rows and codes, D / 32 bytes of scales at once
  const int sb = head_dim / 32;
  if (stride_q_token % 8 || stride_q_head % 8 || !aligned(q, 16) || !aligned(codes, 16) || !aligned(scales, uintptr_t(sb)))
    return FXPR_E_ARG;
  // (the kernels multiply a block index by a 32-bit stride, and keep a page's
  // rows within 32-bit offsets)
  for (int64_t s : {stride_codes_block, stride_codes_half, stride_codes_slot, stride_codes_head})
    if (s % 16 || s < 0 || s > int64_t(0xffffffff)) return FXPR_E_ARG;
  for (int64_t s : {stride_scales_block, stride_scales_half, stride_scales_slot, stride_scales_head})
    if (s % sb || s < 0 || s > int64_t(0xffffffff)) return FXPR_E_ARG;
  if (std::max(stride_codes_slot, stride_scales_slot) * 16 > int64_t(0x7fffffff) ||
      std::max(stride_codes_head, stride_scales_head) * num_kv_heads > int64_t(0xffffffff))
    return FXPR_E_ARG;
  if (int64_t(max_blocks_per_seq) * page_size > int64_t(0x7fffffff) - 1024) return FXPR_E_SHAPE;
  const int64_t slots = chunk_slots(max_blocks_per_seq, page_size);
  const int64_t max_rows = int64_t(max_query_len > 1 ? max_query_len : 1) * (num_heads / num_kv_heads);
  Planned plan = plan_mx4(num_requests, num_tokens, num_heads, num_kv_heads, head_dim, page_size, max_query_len,
                          max_blocks_per_seq, std::max(window_size, 0), int_bits, num_kv_splits);
  // (quotient()'s ranges: rows of a request by the group, request x kv head by
  // the kv heads)
  const int64_t group = num_heads / num_kv_heads;
  if ((std::max(max_rows, num_tokens * group) + 2 * PQROWS * (int64_t(num_requests) + 1)) * group > int64_t(0xffffffff) ||
      int64_t(num_requests) * num_kv_heads * num_kv_heads > int64_t(0xffffffff))
    return FXPR_E_SHAPE;
  if (max_rows > int64_t(0x7fffffff) ||
      (num_tokens * group / PQROWS + num_requests) * num_kv_heads > int64_t(0x7fffffff))
    return FXPR_E_SHAPE;
  if (plan.ws.total > 0 && (!workspace || workspace_bytes < plan.ws.total || !aligned(workspace, 16)))
    return FXPR_E_WORKSPACE;

  Mx4Args m{};
  AttnArgs& a = m.a;
  m.kc = static_cast<const uint8_t*>(codes);
  m.vc = m.kc + stride_codes_half;
  m.ks = static_cast<const uint8_t*>(scales);
  m.vs = m.ks + stride_scales_half;
  m.c_blk = uint32_t(stride_codes_block);
  m.c_slot = uint32_t(stride_codes_slot);
  m.c_head = uint32_t(stride_codes_head);
  m.s_blk = uint32_t(stride_scales_block);
  m.s_slot = uint32_t(stride_scales_slot);
  m.s_head = uint32_t(stride_scales_head);
  m.by_group = reciprocal(uint32_t(num_heads / num_kv_heads));
  m.by_heads = reciprocal(uint32_t(num_kv_heads));
  m.by_reqs = reciprocal(uint32_t(num_requests));
  a.q = q;
  a.o = o;
  a.qsl = query_start_loc;
  a.seq_lens = seq_lens;
  a.bt = block_table;
  a.alibi = alibi_slopes;
  char* base = static_cast<char*>(workspace);
  if (plan.ws.total > 0) {
    a.crange = reinterpret_cast<int*>(base + plan.ws.crange);
    a.pmax = reinterpret_cast<float*>(base + plan.ws.pmax);
    a.den_ws = base + plan.ws.den;
    a.wv_ws = base + plan.ws.wv;
  }
  a.chunk_slots = int(slots);
  a.sq_t = stride_q_token;
  a.sq_h = stride_q_head;
  a.so_t = stride_o_token;
  a.so_h = stride_o_head;
  a.sbt = stride_bt_row;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.window = window_size > 0 ? window_size : 0;
  a.causal = is_causal ? 1 : 0;
  a.max_blocks = max_blocks_per_seq;
  a.num_requests = num_requests;
  a.num_blocks = num_blocks;
  a.num_tokens = num_tokens;
  a.lmax = int64_t(max_blocks_per_seq) * page_size;
  a.ps_shift = __builtin_ctz(unsigned(page_size));
  a.scale_log2 = softmax_scale_log2;
  a.softcap_log2 = softcap_log2;
  a.fxp_scale = pow2f(frac_bits);
  a.fxp_inv = pow2f(-frac_bits);
  m.vlim = (int_bits == 16 ? 32767.0f : 4194304.0f) * a.fxp_inv;
  hipStream_t st = as_stream(stream);
  return io_dtype == FXPR_DTYPE_BF16 ? run_mx4_bf16(m, plan.p, int_bits, num_requests, max_query_len, num_tokens, st)
                                     : run_mx4_f16(m, plan.p, int_bits, num_requests, max_query_len, num_tokens, st);
}
