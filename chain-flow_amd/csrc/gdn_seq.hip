// The gated delta rule over committed tokens on MI355X: the recurrent step of a decode batch and the rule
// over whole prefill chunks, in the layout, with the gates and the state slots of the serving tree form
// (gdn.hip): value head hv of a row of mixed_qkv [T][2 H K + HV V] uses q/k head hv / (HV / H),
//     g = -exp(A_log) softplus(a + dt_bias),  beta = bf16(sigmoid(b)),
//     S = e^g S;  d = beta (v - S k^);  S += d k^T;  o = S q^
// with k^ = k / sqrt(|k|^2 + 1e-6), q^ = scale q / sqrt(|q|^2 + 1e-6) and S a slot [V][K] of the state.
// The state is carried in fp32 and rounded to the slot's type once, at the end of the call.
#include "cfh_gdn.h"
#include "cfh_host.h"

namespace {

struct GdnSeqArgs {
  const uint16_t* qkv;   // [T][ld] bf16
  const uint16_t* ga;    // [T][HV] bf16
  const uint16_t* gb;    // [T][HV] bf16
  const float* A_log;    // [HV]
  const float* dt_bias;  // [HV]
  void* state;           // [nslots][HV][V][K]
  const int* slots;      // [S]
  const int* cu;         // [S + 1], or null: sequence s is row s
  const uint8_t* initial;  // [S] or null: 0 = start from zero instead of the slot
  uint16_t* out;         // [T][HV][V] bf16
  int* status;
  int T, S, H, HV, V, ld, nslots, l2norm;
  float scale;
};

// softplus by log1p: with log(1 + exp(x)) a decay near 1 (x below -5, the usual ones) keeps few digits of its
// logarithm, which thousands of tokens add up.
__device__ __forceinline__ void seq_gates(float x, float Aexp, float b, float& g, float& beta) {
  g = -Aexp * (x <= 20.0f ? log1pf(expf(x)) : x);
  const float t = expf(-fabsf(b));             // (e^-b overflows below -88, where the sigmoid is still a number)
  beta = round_bf16((b < 0.f ? t : 1.0f) / (1.0f + t));
}

// Whether sequence s may use its slot: 1 yes, 0 a padding entry (slot -1), -1 refused (outside the state, or
// shared with another sequence, whose updates would race).  Uniform over the wave.
__device__ __forceinline__ int slot_verdict(const int* slots, int S, int s, int nslots) {
  const int mine = slots[s], lane = threadIdx.x & 63;
  if (mine == -1) return 0;
  int same = 0;
  for (int i = lane; i < S; i += 64) same += i != s && slots[i] == mine;
  return (__ballot(same > 0) || mine < 0 || mine >= nslots) ? -1 : 1;
}

// The simplest form, and the decode step: a wave takes 16 value rows of one (sequence, value head) and its
// tokens one after another.  Lane 16 g + p holds an 8-element share of K of rows 4 g + (0..3) (cfh_gdn.h);
// a dot product is 8 products and a 16-lane DPP sum.  No LDS and no barrier.
template <typename T>
__global__ void __launch_bounds__(64) k_gdn_rows(GdnSeqArgs a) {
  constexpr int NR = sizeof(T) / 2;
  const int nvs = a.V / 16;
  int u = blockIdx.x;
  const int vs = u % nvs;
  u /= nvs;
  const int hv = u % a.HV, s = u / a.HV;
  const int lane = threadIdx.x, p = lane & 15, r0 = vs * 16 + (lane >> 4) * 4;
  const int t0 = a.cu ? a.cu[s] : s, t1 = a.cu ? a.cu[s + 1] : s + 1;
  const int ok = slot_verdict(a.slots, a.S, s, a.nslots);
  const bool rows = t0 >= 0 && t1 <= a.T && t0 <= t1;
  if (ok == 0) return;
  if (ok < 0 || !rows) {
    if (a.status && lane == 0) a.status[0] = 1;
    if (rows)
      for (int t = t0; t < t1; ++t)
        if (p < 4) a.out[((size_t)t * a.HV + hv) * a.V + r0 + p] = 0x7fc0;
    return;
  }
  if (t0 == t1) return;
  T* const st = (T*)a.state + (((size_t)a.slots[s] * a.HV + hv) * a.V + r0) * GDN_DK;
  float S[4][8];
  uint4 raw[4][NR];
  if (!a.initial || a.initial[s]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) row_load(st + i * GDN_DK, p, raw[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) row_widen(raw[i], S[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) S[i][x] = 0.f;
  }
  const float Aexp = expf(a.A_log[hv]), dtb = a.dt_bias[hv];
  const int h = hv / (a.HV / a.H);
  const size_t qo = (size_t)h * GDN_DK, ko = ((size_t)a.H + h) * GDN_DK;
  const size_t vo = 2 * (size_t)a.H * GDN_DK + (size_t)hv * a.V + r0;
  for (int t = t0; t < t1; ++t) {
    const uint16_t* row = a.qkv + (size_t)t * a.ld;
    // the lane's share of k and q, in the order of its share of the state's rows
    float k[8], q[8], v[4], g, beta;
    uint2 kw[2], qw[2];
    const int x0 = sizeof(T) == 2 ? 8 * p : 4 * p, x1 = sizeof(T) == 2 ? 8 * p + 4 : 64 + 4 * p;
    kw[0] = *(const uint2*)(row + ko + x0); kw[1] = *(const uint2*)(row + ko + x1);
    qw[0] = *(const uint2*)(row + qo + x0); qw[1] = *(const uint2*)(row + qo + x1);
    const uint2 vw = *(const uint2*)(row + vo);
    const size_t m = (size_t)t * a.HV + hv;
    seq_gates(bf16f(a.ga[m]) + dtb, Aexp, bf16f(a.gb[m]), g, beta);
    const float e = expf(g);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[4 * i] = __uint_as_float(kw[i].x << 16); k[4 * i + 1] = __uint_as_float(kw[i].x & 0xffff0000u);
      k[4 * i + 2] = __uint_as_float(kw[i].y << 16); k[4 * i + 3] = __uint_as_float(kw[i].y & 0xffff0000u);
      q[4 * i] = __uint_as_float(qw[i].x << 16); q[4 * i + 1] = __uint_as_float(qw[i].x & 0xffff0000u);
      q[4 * i + 2] = __uint_as_float(qw[i].y << 16); q[4 * i + 3] = __uint_as_float(qw[i].y & 0xffff0000u);
    }
    v[0] = __uint_as_float(vw.x << 16); v[1] = __uint_as_float(vw.x & 0xffff0000u);
    v[2] = __uint_as_float(vw.y << 16); v[3] = __uint_as_float(vw.y & 0xffff0000u);
    float rk = 1.f, rq = a.scale;
    if (a.l2norm) {
      float kk = 0.f, qq = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) { kk += k[x] * k[x]; qq += q[x] * q[x]; }
      rk = 1.0f / sqrtf(row_sum(kk) + 1e-6f);
      rq = a.scale / sqrtf(row_sum(qq) + 1e-6f);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) { k[x] *= rk; q[x] *= rq; }
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float d0 = 0.f, d1 = 0.f;
#pragma unroll
      for (int x = 0; x < 8; x += 2) {
        S[i][x] *= e; S[i][x + 1] *= e;
        d0 += S[i][x] * k[x]; d1 += S[i][x + 1] * k[x + 1];
      }
      const float d = (v[i] - row_sum(d0 + d1)) * beta;
      d0 = d1 = 0.f;
#pragma unroll
      for (int x = 0; x < 8; x += 2) {
        S[i][x] += k[x] * d; S[i][x + 1] += k[x + 1] * d;
        d0 += S[i][x] * q[x]; d1 += S[i][x + 1] * q[x + 1];
      }
      o[i] = row_sum(d0 + d1);
    }
    const float mine = p & 2 ? (p & 1 ? o[3] : o[2]) : (p & 1 ? o[1] : o[0]);
    if (p < 4) a.out[m * a.V + r0 + p] = to_bf16(mine);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    row_pack(S[i], raw[i]);
    row_store(st + i * GDN_DK, p, raw[i]);
  }
}

constexpr int GDN_SEQS = 4096;   // sequences a call (every wave looks for its slot among theirs)

int seq_args(GdnSeqArgs& g, const void* mixed_qkv, const void* a, const void* b, const float* A_log,
             const float* dt_bias, void* ssm_state, int nslots, const int32_t* slots, int S, int T, int H, int HV, int K,
             int V, int use_l2norm, float scale, void* out, int32_t* status) {
  if (T < 0 || S < 0 || H < 1 || HV < H || HV % H || V < 16 || V % 16 || nslots < 1) return CFH_E_INVALID;
  if (K != GDN_DK || S > GDN_SEQS) return CFH_E_UNSUPPORTED;
  if (T == 0 || S == 0) return CFH_OK;
  if (!mixed_qkv || !a || !b || !A_log || !dt_bias || !ssm_state || !slots || !out) return CFH_E_INVALID;
  if (((uintptr_t)mixed_qkv | (uintptr_t)ssm_state) % 16 || (uintptr_t)out % 2) return CFH_E_INVALID;
  g.qkv = (const uint16_t*)mixed_qkv; g.ga = (const uint16_t*)a; g.gb = (const uint16_t*)b; g.A_log = A_log;
  g.dt_bias = dt_bias; g.state = ssm_state; g.slots = slots; g.out = (uint16_t*)out; g.status = status; g.T = T;
  g.S = S; g.H = H; g.HV = HV; g.V = V; g.ld = 2 * H * K + HV * V; g.nslots = nslots; g.l2norm = use_l2norm ? 1 : 0;
  g.scale = scale;
  return CFH_OK;
}

int launch_rows(const GdnSeqArgs& g, int state_bf16, hipStream_t st) {
  const long long blocks = (long long)g.S * g.HV * (g.V / 16);
  if (blocks > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  if (state_bf16) hipLaunchKernelGGL(k_gdn_rows<uint16_t>, dim3((unsigned)blocks), dim3(64), 0, st, g);
  else hipLaunchKernelGGL(k_gdn_rows<float>, dim3((unsigned)blocks), dim3(64), 0, st, g);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // namespace

extern "C" {

int cfh_gdn_decode(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                   void* ssm_state, int state_bf16, int nslots, const int32_t* slots, int S, int H, int HV, int K, int V,
                   int use_l2norm, float scale, void* out, int32_t* status, void* stream) {
  GdnSeqArgs g = {};
  if (int rc = seq_args(g, mixed_qkv, a, b, A_log, dt_bias, ssm_state, nslots, slots, S, S, H, HV, K, V, use_l2norm,
                        scale, out, status))
    return rc;
  if (S == 0) return CFH_OK;
  return launch_rows(g, state_bf16, (hipStream_t)stream);
}

int64_t cfh_gdn_prefill_ws_bytes(int T, int S, int HV) {
  if (T < 0 || S < 0 || HV < 1) return -1;
  return 0;
}

int cfh_gdn_prefill(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                    void* ssm_state, int state_bf16, int nslots, const int32_t* slots, const int32_t* cu_seqlens,
                    const uint8_t* initial, int S, int T, int H, int HV, int K, int V, int use_l2norm, float scale,
                    void* out, void* ws, int32_t* status, void* stream) {
  GdnSeqArgs g = {};
  if (int rc = seq_args(g, mixed_qkv, a, b, A_log, dt_bias, ssm_state, nslots, slots, S, T, H, HV, K, V, use_l2norm,
                        scale, out, status))
    return rc;
  if (S == 0 || T == 0) return CFH_OK;
  if (!cu_seqlens) return CFH_E_INVALID;
  g.cu = cu_seqlens;
  g.initial = initial;
  return launch_rows(g, state_bf16, (hipStream_t)stream);
}

}  // extern "C"
