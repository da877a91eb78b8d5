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
// the elements end at 240 (off by up to 15.9 scales, less than 2^-4 of the value), so that every finite value reads back
// finite.
#include "cfh_host.h"
#include "cfh_kv.h"

namespace {

// Groups of D / 8 lanes take the key and the value of one (row, head), 8 elements a lane: 16-byte accesses of the
// 2-byte side, 8-byte ones of the 8-bit side; N of them a group, their loads in flight together.
//   Bound by memory: 16,000 rows of 4 heads of 256 into an 8-bit cache (98 MB, scattered slots) 20.4 us, 4.8 TB/s; 40,000
// such rows back (246 MB) 48.5 us, 5.1 TB/s, as a copy of 1 GiB (where every call writes the same 164 MB, which the
// last cache partly holds, 41).  32 rows: 3.5 us, a launch.
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

typedef unsigned v4u __attribute__((ext_vector_type(4)));   // (arrays of uint4, a union, went to memory here)

template <bool BF, bool F8, int D, int N>
__global__ void __launch_bounds__(256) k_kv_write(KvRowsArgs a) {
  constexpr int L = D / 8, R = 256 / L;      // lanes a row, rows a workgroup and pass
  const int c = threadIdx.x % L;
  const unsigned rows = (unsigned)a.T * a.Hkv;
  v4u kr[N], vr[N];
  unsigned h[N];
  int slot[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned r = (blockIdx.x * N + i) * R + threadIdx.x / L, rc = min(r, rows - 1);
    const unsigned t = rc / a.Hkv;
    h[i] = rc - t * a.Hkv;
    slot[i] = r < rows ? a.slots[t] : -1;
    kr[i] = *(const v4u*)(a.key + (size_t)t * a.ld_k + h[i] * D + c * 8);
    vr[i] = *(const v4u*)(a.value + (size_t)t * a.ld_v + h[i] * D + c * 8);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {              // (whole groups take a branch: the DPP steps stay within one)
    if (slot[i] < 0 || slot[i] >= a.slots_all) {
      if (slot[i] >= a.slots_all && a.status && c == 0) a.status[0] = 1;
      continue;
    }
    const unsigned blk = (unsigned)slot[i] / a.page, at = slot[i] - blk * a.page;
    const unsigned in = (at * a.Hkv + h[i]) * D + c * 8;
    auto put = [&](v4u raw, void* cache, long long bs, uint8_t* ex) {
      const size_t dst = (size_t)blk * bs + in;
      if constexpr (!F8) {
        *(v4u*)((u16*)cache + dst) = raw;
      } else {
        float x[8];
        widen8<BF>(make_uint4(raw[0], raw[1], raw[2], raw[3]), x);
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
        *(uint2*)((uint8_t*)cache + dst) = w;
        if (c == 0) ex[(size_t)slot[i] * a.Hkv + h[i]] = (uint8_t)code;
      }
    };
    put(kr[i], a.kc, a.bs_k, a.ke);
    put(vr[i], a.vc, a.bs_v, a.ve);
  }
}

template <bool BF, bool F8, int D, int N>
__global__ void __launch_bounds__(256) k_kv_read(KvRowsArgs a) {
  constexpr int L = D / 8, R = 256 / L;
  const int c = threadIdx.x % L;
  const unsigned rows = (unsigned)a.T * a.Hkv;
  unsigned r[N], h[N];
  int slot[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i] = (blockIdx.x * N + i) * R + threadIdx.x / L;
    const unsigned rc = min(r[i], rows - 1), t = rc / a.Hkv;
    h[i] = rc - t * a.Hkv;
    slot[i] = a.slots[t];
  }
  uint4 out[N][2];
  int code[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = slot[i] >= 0 && slot[i] < a.slots_all;
    if (!in && slot[i] >= 0 && a.status && c == 0) a.status[0] = 1;
    const unsigned s = in ? slot[i] : 0, blk = s / a.page;   // (a slot outside the cache: any row, cleared below)
    const unsigned off = ((s - blk * a.page) * a.Hkv + h[i]) * D + c * 8;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const size_t src = (size_t)blk * (v ? a.bs_v : a.bs_k) + off;
      if constexpr (F8) {
        const uint2 w = *(const uint2*)((const uint8_t*)(v ? a.vc : a.kc) + src);
        out[i][v] = make_uint4(w.x, w.y, 0, 0);
        code[i][v] = (v ? a.ve : a.ke)[(size_t)s * a.Hkv + h[i]];
      } else {
        out[i][v] = *(const uint4*)((const u16*)(v ? a.vc : a.kc) + src);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (r[i] >= rows) break;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint4 o = out[i][v];
      if constexpr (F8) o = dequant8<BF>(make_uint2(o.x, o.y), code[i][v]);
      if (slot[i] < 0 || slot[i] >= a.slots_all) o = make_uint4(0, 0, 0, 0);
      *(uint4*)((v ? a.out_value : a.out_key) + (size_t)r[i] * D + c * 8) = o;
    }
  }
}

// Rows a group: four where that still makes WIDE workgroups, else one.
constexpr int WIDE = 1024;
template <typename F>
int launch_rows_of(long long rows, int D, F launch) {
  const long long per = 256 / (D / 8), wgs = (rows + per - 1) / per;
  if (rows > 0x3fffffffll) return CFH_E_UNSUPPORTED;
  if (wgs >= 4 * WIDE) launch(std::integral_constant<int, 4>{}, (unsigned)((wgs + 3) / 4));
  else launch(std::integral_constant<int, 1>{}, (unsigned)wgs);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int rows_ok(const KvRowsArgs& a, int D, int blocks, bool f8) {
  if (a.T < 0 || a.Hkv < 1 || blocks < 1 || a.page < 1) return CFH_E_INVALID;
  if (D != 64 && D != 128 && D != 256) return CFH_E_UNSUPPORTED;
  if (a.slots_all > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  if (!a.kc || !a.vc || (f8 && (!a.ke || !a.ve))) return CFH_E_INVALID;
  const long long inner = (long long)a.page * a.Hkv * D;
  if (inner > 0x7fffffffll) return CFH_E_UNSUPPORTED;
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
  int rc = CFH_OK;
  kv_dispatch(is_bf16, f8, D, [&](auto bf, auto q, auto d) {
    rc = launch_rows_of((long long)T * Hkv, D, [&](auto n, unsigned grid) {
      hipLaunchKernelGGL((k_kv_write<bf.value, q.value, d.value, n.value>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    });
  });
  return rc;
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
  int rc = CFH_OK;
  kv_dispatch(is_bf16, f8, D, [&](auto bf, auto q, auto d) {
    rc = launch_rows_of((long long)T * Hkv, D, [&](auto n, unsigned grid) {
      hipLaunchKernelGGL((k_kv_read<bf.value, q.value, d.value, n.value>), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    });
  });
  return rc;
}

}  // extern "C"
