// Attention of new rows over a paged cache on MI355X: a prefill chunk, a decode step's single rows, or the
// nodes of draft trees over the committed prefix.
//
// Sequence s has the query rows cu_q[s] .. cu_q[s + 1] and seq_lens[s] tokens in its pages table[s][..].
// Its row i of n sees token j where j < len and, if causal, j <= len - n + i (the chunk's own rows are the
// cache's last ones).  Head h reads kv head h / (H / Hkv).
//     o = sum_j softmax_j(scale q.k_j) v_j,   lse = log sum_j exp(scale q.k_j)
// A row that sees nothing gives o = 0 and lse = -inf.
#include "cfh_host.h"
#include "cfh_kv.h"

namespace {

struct PagedArgs {
  const u16* q;                // [T][H][D], row stride q_ld
  u16* out;                    // [T][H][D], row stride o_ld
  float* lse;                  // [H][T]
  const void* kc; const void* vc;
  const uint8_t* ke; const uint8_t* ve;
  const int* table;            // [S][table_ld]
  const int* lens;             // [S]
  const int* cu;               // [S + 1]
  int* status;
  long long q_ld, o_ld, bs_k, bs_v;
  int T, H, Hkv, S, blocks, page, table_ld, max_blocks, causal;
  float scale;
};

// Whether a sequence's rows lie in the query.
__device__ __forceinline__ bool bounds_ok(const PagedArgs& a, int c0, int c1) { return c0 >= 0 && c0 <= c1 && c1 <= a.T; }

// The simplest form: a wave per (row, head), lane l the elements l * EPL .., one token after another with
// the running maximum and sum of the softmax.
template <bool BF, bool F8, int D>
__global__ void __launch_bounds__(256) k_paged_rows(PagedArgs a) {
  constexpr int EPL = D / 64;
  const int lane = threadIdx.x & 63;
  const long long gw = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t = (int)(gw / a.H), h = (int)(gw - (long long)t * a.H);
  if (a.status && gw == 0)
    for (int i = lane; i < a.S; i += 64)
      if (!bounds_ok(a, a.cu[i], a.cu[i + 1])) a.status[0] = 1;
  if (t >= a.T) return;
  int lo = 0, hi = a.S;                         // the first i >= 1 with cu[i] > t, less one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int s = lo, c0 = a.cu[s], c1 = a.cu[s + 1];
  if (t < c0 || t >= c1 || !bounds_ok(a, c0, c1)) return;   // a row of no sequence
  const int hk = h / (a.H / a.Hkv);
  int len = a.lens[s];
  const long long most = (long long)a.max_blocks * a.page;
  bool bad = len < 0 || len > most;
  len = bad ? 0 : len;
  const int vis = a.causal ? min(len, len - (c1 - c0) + (t - c0) + 1) : len;
  float q[EPL], acc[EPL], m = -INFINITY, l = 0.f;
  auto ld = [&](const void* p, size_t i) {
    if constexpr (BF) return __uint_as_float((unsigned)((const u16*)p)[i] << 16);
    else return (float)__builtin_bit_cast(_Float16, ((const u16*)p)[i]);
  };
  for (int e = 0; e < EPL; ++e) {
    q[e] = ld(a.q, (size_t)t * a.q_ld + (size_t)h * D + lane * EPL + e);
    acc[e] = 0.f;
  }
  for (int j = 0; j < vis; ++j) {
    const int b = j / a.page, at = j - b * a.page;
    const int blk = a.table[(size_t)s * a.table_ld + b];
    if (blk < 0 || blk >= a.blocks) { bad = true; break; }
    auto row = [&](const void* c, const uint8_t* ex, long long bs, float (&x)[EPL]) {
      const size_t i = (size_t)blk * bs + ((size_t)at * a.Hkv + hk) * D + lane * EPL;
      for (int e = 0; e < EPL; ++e) {
        if constexpr (F8) {
          const float sc = __uint_as_float((unsigned)ex[((size_t)blk * a.page + at) * a.Hkv + hk] << 23);
          const f32x2k v = __builtin_amdgcn_cvt_pk_f32_fp8((int)((const uint8_t*)c)[i + e], false);
          const unsigned w = pack2<BF>(v[0] * sc, 0.f);
          x[e] = ld(&w, 0);
        } else {
          x[e] = ld(c, i + e);
        }
      }
    };
    float k[EPL], v[EPL], d = 0.f;
    row(a.kc, a.ke, a.bs_k, k);
    row(a.vc, a.ve, a.bs_v, v);
    for (int e = 0; e < EPL; ++e) d += q[e] * k[e];
    const float x = wave_sum(d) * a.scale;
    const float mn = fmaxf(m, x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float w = expf(m - base), p = expf(x - base);
    l = l * w + p;
    for (int e = 0; e < EPL; ++e) acc[e] = acc[e] * w + p * v[e];
    m = mn;
  }
  float inv = l == 0.f ? 0.f : 1.f / l, lse = l == 0.f ? -INFINITY : m + logf(l);
  if (bad) {
    inv = lse = __builtin_nanf("");
    if (a.status && lane == 0) a.status[0] = 1;
  }
  for (int e = 0; e < EPL; ++e)
    a.out[(size_t)t * a.o_ld + (size_t)h * D + lane * EPL + e] = (u16)pack2<BF>(acc[e] * inv, 0.f);
  if (lane == 0) a.lse[(size_t)h * a.T + t] = lse;
}

}  // namespace

extern "C" {

int64_t cfh_paged_attn_ws_bytes(int T, int H, int Hkv, int D, int S, int max_len) {
  if (T < 0 || H < 1 || Hkv < 1 || H % Hkv || S < 0 || max_len < 0) return -1;
  return 0;
}

int cfh_paged_attn(const void* q, long long q_ld, int T, int H, int Hkv, int D, int is_bf16, const void* k_cache,
                   long long bs_k, const void* v_cache, long long bs_v, const uint8_t* k_exp, const uint8_t* v_exp,
                   int blocks, int page, const int32_t* table, int table_ld, int max_blocks, const int32_t* seq_lens,
                   const int32_t* cu_q, int S, float scale, int causal, int max_len, void* out, long long o_ld,
                   float* lse, void* ws, int32_t* status, void* stream) {
  if (T < 0 || S < 0 || H < 1 || Hkv < 1 || H % Hkv || blocks < 1 || page < 1 || max_blocks < 0 ||
      table_ld < max_blocks || max_len < 0)
    return CFH_E_INVALID;
  if (D != 64 && D != 128 && D != 256) return CFH_E_UNSUPPORTED;
  if ((long long)blocks * page > 0x7fffffffll || (long long)max_blocks * page > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  const bool f8 = k_exp || v_exp;
  if (!k_cache || !v_cache || (f8 && (!k_exp || !v_exp))) return CFH_E_INVALID;
  const long long inner = (long long)page * Hkv * D;
  if (bs_k < inner || bs_v < inner || bs_k % 16 || bs_v % 16 || ((uintptr_t)k_cache | (uintptr_t)v_cache) % 16)
    return CFH_E_INVALID;
  if (T == 0 || S == 0) return CFH_OK;
  if (!q || !out || !lse || !seq_lens || !cu_q || (max_blocks && !table) || q_ld < (long long)H * D ||
      o_ld < (long long)H * D || q_ld % 8 || o_ld % 8 || ((uintptr_t)q | (uintptr_t)out) % 16)
    return CFH_E_INVALID;
  PagedArgs a = {};
  a.q = (const u16*)q; a.out = (u16*)out; a.lse = lse; a.kc = k_cache; a.vc = v_cache; a.ke = k_exp; a.ve = v_exp;
  a.table = table; a.lens = seq_lens; a.cu = cu_q; a.status = status; a.q_ld = q_ld; a.o_ld = o_ld; a.bs_k = bs_k;
  a.bs_v = bs_v; a.T = T; a.H = H; a.Hkv = Hkv; a.S = S; a.blocks = blocks; a.page = page; a.table_ld = table_ld;
  a.max_blocks = max_blocks; a.causal = causal ? 1 : 0; a.scale = scale;
  const long long waves = (long long)T * H;
  const dim3 grid((unsigned)((waves + 3) / 4));
  hipStream_t st = (hipStream_t)stream;
  kv_dispatch(is_bf16, f8, D, [&](auto bf, auto e8, auto d) {
    hipLaunchKernelGGL((k_paged_rows<bf.value, e8.value, d.value>), grid, dim3(256), 0, st, a);
  });
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // extern "C"
