// The paged key / value cache of the target's attention layers on MI355X: rows written into slots
// (copied, or quantised to 8 bits as they are written) and read back.
//
// Slot n of a cache [blocks][page][Hkv][D] is row n % page of block n / page.  An 8-bit cache holds e4m3
// elements and one byte c per (slot, head) that stands for the scale 2^(c - 127):
//     c - 127 = the least E >= -126 with amax <= 448 * 2^E   (amax: the row's largest finite magnitude)
//     element = rne_e4m3(x / 2^E)
// A power of two divides exactly, so the rounding to e4m3 is the only one (at most half a step, 2^-4 of
// the value while it is normal in e4m3), reading back multiplies exactly, and a value next to a rounding
// border cannot fall to its other side.  It costs no precision: e4m3's relative step is the same in every
// binade, and the up to one binade left unused at the top is one of 15.  The format has no infinity:
// NaN and infinite elements are stored as NaN.  Where 256 * 2^E is above the source type's largest value
// the elements end at 240 (still within half a step), so that every finite value reads back finite.
#include "cfh_host.h"
#include "cfh_kv.h"

namespace {

// Groups of D / 8 lanes take one (row, head) each, 8 elements a lane: 16-byte accesses of the 2-byte side,
// 8-byte ones of the 8-bit side.  Keys and values are the two halves of one launch.
struct KvRowsArgs {
  const u16* key; const u16* value;          // [T][Hkv][D], row strides ld_k / ld_v
  u16* out_key; u16* out_value;              // (reading)
  void* kc; void* vc;                        // [blocks][page][Hkv][D], block strides in elements
  uint8_t* ke; uint8_t* ve;                  // [blocks][page][Hkv] or null
  const int* slots;                          // [T]
  int* status;
  long long ld_k, ld_v, bs_k, bs_v;
  long long slots_all;                       // blocks * page
  int T, Hkv, page;
};

// The largest of v over the L lanes of the group (L = 8, 16 or 32).
template <int L>
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp_f32<DPP_XOR1>(v));
  v = fmaxf(v, dpp_f32<DPP_XOR2>(v));
  v = fmaxf(v, dpp_f32<DPP_HMIRROR>(v));
  if constexpr (L >= 16) v = fmaxf(v, dpp_f32<DPP_MIRROR>(v));
  if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16));
  return v;
}

template <bool BF, bool F8, int D>
__global__ void __launch_bounds__(256) k_kv_write(KvRowsArgs a) {
  constexpr int L = D / 8, R = 256 / L;      // lanes a row, rows a workgroup
  const long long r = (long long)blockIdx.x * R + threadIdx.x / L;
  const int c = threadIdx.x % L;
  const bool val = blockIdx.y;
  const int t = (int)(r / a.Hkv), h = (int)(r - (long long)t * a.Hkv);
  if (t >= a.T) return;                      // (whole groups: the DPP steps stay within one)
  const int slot = a.slots[t];
  const u16* src = (val ? a.value : a.key) + t * (val ? a.ld_v : a.ld_k) + (size_t)h * D + c * 8;
  const uint4 raw = *(const uint4*)src;
  if (slot < 0 || slot >= a.slots_all) {
    if (slot >= a.slots_all && a.status && c == 0) a.status[0] = 1;
    return;
  }
  const int blk = slot / a.page, at = slot - blk * a.page;
  const size_t dst = (size_t)blk * (val ? a.bs_v : a.bs_k) + ((size_t)at * a.Hkv + h) * D + c * 8;
  if constexpr (!F8) {
    *(uint4*)((u16*)(val ? a.vc : a.kc) + dst) = raw;
  } else {
    float x[8];
    widen8<BF>(raw, x);
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
    const unsigned u = __float_as_uint(group_max<L>(m));
    // 448 = 1.75 * 2^8: the biased exponent less 8, one more where the mantissa is above 1.75
    const int code = max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u), 1);
    const float inv = __uint_as_float((unsigned)(254 - code) << 23);
    const float most = code == (BF ? 247 : 135) ? 240.f : 448.f;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = fminf(fmaxf(x[e] * inv, -most), most);
      if (!(fabsf(x[e]) < INFINITY)) y[e] = __builtin_nanf("");
    }
    uint2 w;
    w.x = pack_e4m3(y[0], y[1], y[2], y[3]);
    w.y = pack_e4m3(y[4], y[5], y[6], y[7]);
    *(uint2*)((uint8_t*)(val ? a.vc : a.kc) + dst) = w;
    if (c == 0) (val ? a.ve : a.ke)[(size_t)slot * a.Hkv + h] = (uint8_t)code;
  }
}

template <bool BF, bool F8, int D>
__global__ void __launch_bounds__(256) k_kv_read(KvRowsArgs a) {
  constexpr int L = D / 8, R = 256 / L;
  const long long r = (long long)blockIdx.x * R + threadIdx.x / L;
  const int c = threadIdx.x % L;
  const bool val = blockIdx.y;
  const int t = (int)(r / a.Hkv), h = (int)(r - (long long)t * a.Hkv);
  if (t >= a.T) return;
  const int slot = a.slots[t];
  uint4 out = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < a.slots_all) {
    const int blk = slot / a.page, at = slot - blk * a.page;
    const size_t src = (size_t)blk * (val ? a.bs_v : a.bs_k) + ((size_t)at * a.Hkv + h) * D + c * 8;
    if constexpr (!F8) {
      out = *(const uint4*)((const u16*)(val ? a.vc : a.kc) + src);
    } else {
      const uint2 w = *(const uint2*)((const uint8_t*)(val ? a.vc : a.kc) + src);
      out = dequant8<BF>(w, (val ? a.ve : a.ke)[(size_t)slot * a.Hkv + h]);
    }
  } else if (slot >= 0 && a.status && c == 0) {
    a.status[0] = 1;
  }
  *(uint4*)((val ? a.out_value : a.out_key) + (size_t)r * D + c * 8) = out;
}

int rows_ok(const KvRowsArgs& a, int D, int blocks, bool f8) {
  if (a.T < 0 || a.Hkv < 1 || blocks < 1 || a.page < 1) return CFH_E_INVALID;
  if (D != 64 && D != 128 && D != 256) return CFH_E_UNSUPPORTED;
  if (a.slots_all > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  if (!a.kc || !a.vc || (f8 && (!a.ke || !a.ve))) return CFH_E_INVALID;
  const long long inner = (long long)a.page * a.Hkv * D;
  if (a.bs_k < inner || a.bs_v < inner || a.bs_k % 16 || a.bs_v % 16) return CFH_E_INVALID;
  if (((uintptr_t)a.kc | (uintptr_t)a.vc) % 16) return CFH_E_INVALID;
  return CFH_OK;
}

}  // namespace

extern "C" {

int cfh_kv_write(const void* key, long long ld_k, const void* value, long long ld_v, int T, int Hkv, int D, int is_bf16,
                 void* k_cache, long long bs_k, void* v_cache, long long bs_v, uint8_t* k_exp, uint8_t* v_exp,
                 int blocks, int page, const int32_t* slots, int32_t* status, void* stream) {
  KvRowsArgs a = {};
  a.key = (const u16*)key; a.value = (const u16*)value; a.kc = k_cache; a.vc = v_cache; a.ke = k_exp; a.ve = v_exp;
  a.slots = slots; a.status = status; a.ld_k = ld_k; a.ld_v = ld_v; a.bs_k = bs_k; a.bs_v = bs_v;
  a.slots_all = (long long)blocks * page; a.T = T; a.Hkv = Hkv; a.page = page;
  const bool f8 = k_exp || v_exp;
  if (int rc = rows_ok(a, D, blocks, f8)) return rc;
  if (T == 0) return CFH_OK;
  if (!key || !value || !slots || ld_k < (long long)Hkv * D || ld_v < (long long)Hkv * D || ld_k % 8 || ld_v % 8 ||
      ((uintptr_t)key | (uintptr_t)value) % 16)
    return CFH_E_INVALID;
  const int R = 256 / (D / 8);
  const long long blocks_x = ((long long)T * Hkv + R - 1) / R;
  if (blocks_x > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  const dim3 grid((unsigned)blocks_x, 2);
  hipStream_t st = (hipStream_t)stream;
  kv_dispatch(is_bf16, f8, D, [&](auto bf, auto q, auto d) {
    hipLaunchKernelGGL((k_kv_write<bf.value, q.value, d.value>), grid, dim3(256), 0, st, a);
  });
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int cfh_kv_read(const void* k_cache, long long bs_k, const void* v_cache, long long bs_v, const uint8_t* k_exp,
                const uint8_t* v_exp, int blocks, int page, const int32_t* slots, int T, int Hkv, int D, int is_bf16,
                void* key, void* value, int32_t* status, void* stream) {
  KvRowsArgs a = {};
  a.out_key = (u16*)key; a.out_value = (u16*)value; a.kc = (void*)k_cache; a.vc = (void*)v_cache;
  a.ke = (uint8_t*)k_exp; a.ve = (uint8_t*)v_exp; a.slots = slots; a.status = status; a.bs_k = bs_k; a.bs_v = bs_v;
  a.slots_all = (long long)blocks * page; a.T = T; a.Hkv = Hkv; a.page = page;
  const bool f8 = k_exp || v_exp;
  if (int rc = rows_ok(a, D, blocks, f8)) return rc;
  if (T == 0) return CFH_OK;
  if (!key || !value || !slots || ((uintptr_t)key | (uintptr_t)value) % 16) return CFH_E_INVALID;
  const int R = 256 / (D / 8);
  const long long blocks_x = ((long long)T * Hkv + R - 1) / R;
  if (blocks_x > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  const dim3 grid((unsigned)blocks_x, 2);
  hipStream_t st = (hipStream_t)stream;
  kv_dispatch(is_bf16, f8, D, [&](auto bf, auto q, auto d) {
    hipLaunchKernelGGL((k_kv_read<bf.value, q.value, d.value>), grid, dim3(256), 0, st, a);
  });
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // extern "C"
