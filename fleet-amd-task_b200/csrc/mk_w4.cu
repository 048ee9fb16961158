// mk_w4.cu -- products with 4-bit weights for a batch of tokens: mk_w4_linear (one weight) and
// mk_w4_experts (a layer's routed experts: gate/up, SwiGLU, down projection, weighted sum).
// The format and the laid-out order are in mk_w4.cuh, the kernel in mk_w4_kernel.cuh.
//
// Formulas. linear: out[t] = x[t] W^T (+ residual[t]). experts: out[t] = (residual[t] +) the sum over
// the token's slots s of w[t, s] W2[e] a(t, e), a = silu(g) u, (g, u) = W13[e] x[t], e = ids[t, s]; a
// slot whose id is outside [0, experts) is empty.
//
// What bounds them. A token costs 2 operations per weight and a weight half a byte, so a batch of T
// tokens does 4 T operations a byte: by the numbers the stream of codes bounds a decode batch of up to
// some forty tokens. What it comes to on B200 (a 16 x 128 block of weights a step, per SM): 133
// instructions at 8 columns, 88 of them to make tensor-core operands of the codes (11 per 8 codes:
// three shifts, four AND-ORs, four subtractions), and 8 MMAs; 157 and 16 at 16 columns. Timed with
// parts left out, a step takes instructions / 4 + 2 cycles an MMA (49 cycles modelled, 52 measured at
// 8 columns; 71 and 74 at 16): an SM partition issues nothing beside an mma.sync. The codes of a step
// take 44 cycles at 6.5 TB/s, so a head of 102400 x 2048 reads at 5.3 TB/s within its 25.6 us (107 MB;
// about 5 us are the launch, the first instructions and loads, and the end), 16 tokens take 35 us and
// 32 tokens 54, bound by issue. tcgen05 was built beside it (codes decoded into tensor memory, 128 rows a
// tile, 16 or 32 columns): 48 to 62 us for 9 to 32 tokens, bound by the chain of a tile (decode, store,
// barrier, MMA, commit, read back), and not kept.
//
// The work is a row of sums (a strip: RT tiles of 16 rows, for up to 8 NT columns) times its units of
// 128 values of K. Each CTA (one per SM) takes an equal range of strips, and each warp an equal,
// contiguous range of the CTA's units, wherever strips begin and end in it: the warps finish together
// whatever the sizes, and nothing is synchronised between them until the end of the range, where the
// warp that began a strip adds the parts of the warps after it, in warp order (the result does not
// depend on timing). (Teams of warps on a strip with a barrier each: 31 us for that head.) A warp loads
// its units, which lie one after the other in memory, straight into registers, one or more ahead; a
// cp.async ring in shared memory took as long and more instructions. The activations are either staged
// once in shared memory in the MMA's order, or, where they do not fit, loaded with each unit (xr): 16
// tokens of K 10944 in 13 us, against 27 in blocks of the 6 tokens whose activations fit (an earlier form).
//
// The experts of a small batch (at most 8 tokens) take two launches: gate/up with the tokens as the
// columns of every expert, then the down projection as one long dot product over the selected
// experts' activations, each expert's part scaled by the tokens' weights for it. A larger batch is
// grouped by expert first (plan_kernel), each expert's slots being its columns, and the slots' outputs
// are added afterwards in slot order (combine_kernel). The launches of one call overlap
// (programmatic dependent launches): 24 us instead of 30 for a small layer's four. The intermediate is the sum
// of two BF16 values, which the down projection multiplies one after the other with the same decoded codes: twice its
// MMAs and activations, 4 to 10 % of a call (one 16-bit value: 20.5, 53 and 95 us below).
// Measured, a layer of 66 experts of 2048 x 1408, 8 slots a token: 1 token 21.3 us (36 MB, 5.4 us at the
// copy rate), 8 tokens in groups of 64 with zero points 58 (172 MB of distinct experts, 26 us), 64 tokens 105
// (295 MB, 45 us).
#include <algorithm>

#include "mk_w4_kernel.cuh"

using namespace w4;

namespace {

constexpr int PLAN_COUNTS = 10240;   // 40 KB: all 32 warps count for up to 320 experts, 10 for 1024

// The slots grouped by expert: columns (slots in expert order, an expert's in slot order), col_token,
// slot_col (a slot's column, -1 if empty), and the items of at most tb columns of one expert. One CTA. A
// column's sums are split where its item lies in the CTAs' ranges, so a slot's place among its expert's columns
// has to be the same on every run: each warp counts the experts of a run of consecutive slots, and the
// places are the counts of the warps before it and of the slots before in its own run. (Places in the order
// of atomics: 162 of 200 runs of 64 tokens of 66 experts differed from the first in some results.) The first
// `warps` warps take `chunk` slots each, a multiple of 32.
__global__ void __launch_bounds__(1024) plan_kernel(const int* __restrict__ ids, int n, int s, int experts, int tb, int warps, int chunk,
                                                    int4* items, int* items_n, int* col_token, int* slot_col) {
  extern __shared__ int cnt[];           // [warps][experts]
  __shared__ int first[MAX_EXPERTS];
  start_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lo = warp < warps ? min(warp * chunk, n) : n, hi = min(lo + chunk, n);
  int* mine = cnt + warp * experts;      // (of warps past the last one: not used)
  for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  for (int i = lo + lane; i < hi; i += 32) {
    const int e = ids[i];
    if ((unsigned)e < (unsigned)experts) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = cnt[w * experts + e];
      cnt[w * experts + e] = sum;
      sum += c;
    }
    first[e] = sum;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int cols = 0, its = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + threadIdx.x, c = e < experts ? first[e] : 0, b = (c + tb - 1) / tb;
      int ci = c, bi = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, ci, o), v = __shfl_up_sync(~0u, bi, o);
        if ((int)threadIdx.x >= o) { ci += u; bi += v; }
      }
      const int col0 = cols + ci - c, it0 = its + bi - b;
      if (e < experts) first[e] = col0;
      for (int k = 0; k < b; ++k) items[it0 + k] = make_int4(e, col0 + k * tb, min(tb, c - k * tb), 0);
      cols += __shfl_sync(~0u, ci, 31);
      its += __shfl_sync(~0u, bi, 31);
    }
    if (threadIdx.x == 0) *items_n = its;
  }
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane, e = i < hi ? ids[i] : -1;
    const bool valid = (unsigned)e < (unsigned)experts;
    const uint32_t same = __match_any_sync(~0u, valid ? e : -1), before = same & ((1u << lane) - 1);
    int col = -1;
    if (valid) {
      col = first[e] + mine[e] + __popc(before);
      col_token[col] = i / s;
    }
    if (i < hi) slot_col[i] = col;
    __syncwarp();
    if (valid && before == 0) mine[e] += __popc(same);
    __syncwarp();
  }
}

// out[t] = (residual[t] +) sum over slots, in slot order, of w[t, s] y[column of the slot]
template <class D>
__global__ void __launch_bounds__(256) combine_kernel(const float* y, const int* slot_col, const float* weights, int s, int h,
                                                      const uint16_t* residual, int64_t ldr, uint16_t* out, int64_t ldo) {
  const int tok = blockIdx.x, j = blockIdx.y * 256 + threadIdx.x;
  wait_predecessor();
  if (j >= h) return;
  float v = residual ? D::one_to_f32(residual[(int64_t)tok * ldr + j]) : 0.0f;
  for (int k = 0; k < s; ++k) {
    const int col = slot_col[tok * s + k];
    if (col >= 0) v = fmaf(weights[tok * s + k], y[(int64_t)col * h + j], v);
  }
  out[(int64_t)tok * ldo + j] = D::round(v);
}

int fail(int code, const char* msg) { return mk::set_last_error(code, msg); }

const char* bad_weight(const MkW4* w) {
  if (!w || !w->codes || !w->scales) return "null 4-bit weight";
  if (w->n < 1 || w->k < 1 || w->experts < 1) return "a 4-bit weight has at least one row, value and expert";
  if (w->n > INT32_MAX - UNIT_K || w->k > INT32_MAX - UNIT_K) return "a 4-bit weight's padded rows and values are below 2^31";
  if (w->group != 32 && w->group != 64 && w->group != 128) return "the group size is 32, 64 or 128";
  if (w->dtype != MK_W4_BF16 && w->dtype != MK_W4_FP16) return "the activations are BF16 or FP16";
  if (((uintptr_t)w->codes & 15) || ((uintptr_t)w->scales & 15) || ((uintptr_t)w->zeros & 15))
    return "laid-out codes, scales and zeros start at 16-byte boundaries";
  return nullptr;
}

int units_of(const MkW4* w) { return (w->k + UNIT_K - 1) / UNIT_K; }

void fill(Args& a, const MkW4* w) {
  a.codes = static_cast<const uint8_t*>(w->codes);
  a.scales = static_cast<const uint8_t*>(w->scales);
  a.zeros = static_cast<const uint8_t*>(w->zeros);
  a.units = div_by(units_of(w));
  a.nv = div_by(units_of(w) * 16);
  a.rows = w->n;
  a.k = w->k;
  a.experts = w->experts;
}

// the current device and its SMs
int device_sms(int* device, int* sms) {
  static std::atomic<int> known[MAX_DEVICES];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES)
    return fail(MK_ECUDA, "cudaGetDevice failed or device ordinal out of range");
  int v = known[dev].load(std::memory_order_relaxed);
  if (!v) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return fail(MK_ECUDA, "device attribute");
    known[dev].store(v, std::memory_order_relaxed);
  }
  *device = dev;
  *sms = v;
  return MK_OK;
}

// about `items` items over the SMs; known: exactly that many
int launch_weight(Args& a, const MkW4* w, int64_t items, bool known, bool xr, int sms, cudaStream_t s) {
  const int strips = (w->n + STRIP_ROWS - 1) / STRIP_ROWS;
  // Two tiles a warp share its activations and its loop, one tile spreads few strips over more CTAs (K 2048,
  // one / two tiles: 2048 rows 6.2 / 8.3 us, 8192 rows 8.3 / 9.3, 20000 rows of 8 tokens 14.1 / 13.0)
  const bool two = items * strips >= 2 * sms && !(xr && (a.cols > 8 || a.mode == DOWN || a.mode == DOWN_SMALL)) && a.cols <= MAX_COLS;
  a.strips = div_by(two ? strips : 2 * strips);
  const int grid = (int)(known ? std::min<int64_t>(sms, items * a.strips.d) : sms);
  return w->dtype == MK_W4_BF16 ? launch_bf16(a, w->group, two, xr, grid, s)
                                : launch_fp16(a, w->group, two, xr, grid, s);
}

// 16-bit rows that start at 4-byte boundaries
bool aligned4(const void* p, int64_t ld) { return ((uintptr_t)p & 3) == 0 && ld % 2 == 0; }
bool aligned16(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

struct Plan {   // the workspace of mk_w4_experts, in bytes from its start
  int64_t items, items_n, col_token, slot_col, act, y, bytes;
  int cols, ldact;
  bool small, xr2;      // xr2: the down projection's activations come with its units
};

const char* plan_experts(const MkW4* w13, const MkW4* w2, int64_t t, int64_t s, Plan* p) {
  if (const char* m = bad_weight(w13)) return m;
  if (const char* m = bad_weight(w2)) return m;
  if (w13->dtype != w2->dtype || w13->experts != w2->experts || w13->n % 2 || w13->n / 2 != w2->k || w13->k != w2->n)
    return "W13 [E, 2 I, H] and W2 [E, H, I] do not belong together";
  if (w13->experts > MAX_EXPERTS) return "at most 1024 experts";
  for (const MkW4* w : {w13, w2})
    if ((int64_t)w->experts * (w->n / STRIP_ROWS + 1) * units_of(w) > INT32_MAX / 2) return "the experts have too many weights";
  if (t < 0 || s < 0 || t * s >= (1 << 24)) return "slots (tokens x slots per token) are from 0 to 2^24 - 1";
  p->small = t <= SMALL_T && t * s <= SMALL_SLOTS && fits(units_of(w13), (int)std::max<int64_t>(t, 1));
  p->cols = (int)std::min<int64_t>(std::max<int64_t>(t, 1), GROUPED_COLS);
  while (p->cols > 1 && !fits(units_of(w13), p->cols)) --p->cols;
  if (!fits(units_of(w13), p->cols)) return "rows are too long for the shared memory";
  p->xr2 = p->small || !fits(units_of(w2), 2 * p->cols);
  const int64_t n = std::max<int64_t>(t * s, 1), items = w13->experts + n / p->cols + 1;
  const int64_t most = std::max((std::max(w13->n, w2->n) / 16 + 2) * std::max<int64_t>(units_of(w13), units_of(w2)), (int64_t)1);
  if (items * most > INT32_MAX / 2) return "too many slots times rows";
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
  if (p->small) {
    p->act = take(2 * 2 * n * t * units_of(w2) * UNIT_K);
  } else {
    p->ldact = (w2->k + 7) / 8 * 8;
    p->items_n = take(4);
    p->items = take(16 * items);
    p->col_token = take(4 * n);
    p->slot_col = take(4 * n);
    p->act = take(2 * 2 * n * p->ldact);
    p->y = take(4 * n * w2->n);
  }
  p->bytes = std::max<int64_t>(at, 256);
  return nullptr;
}

}  // namespace

extern "C" int mk_w4_linear(const MkW4* w, const void* x, int64_t ldx, int32_t t, const void* residual, int64_t ldr,
                            void* out, int64_t ldo, int32_t out_f32, void* stream) {
  if (const char* m = bad_weight(w)) return fail(MK_EINVAL, m);
  if (w->experts != 1) return fail(MK_EINVAL, "mk_w4_linear takes one weight");
  if (t < 0) return fail(MK_EINVAL, "a negative number of tokens");
  if (t == 0) return MK_OK;
  if (!x || !out) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)x & 1) || ((uintptr_t)residual & 1) || ((uintptr_t)out & (out_f32 ? 3 : 1)))
    return fail(MK_EINVAL, "misaligned x, residual or out");
  int sms = 0;
  Args a{};
  if (int rc = device_sms(&a.device, &sms)) return rc;
  fill(a, w);
  a.mode = LINEAR;
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  // even blocks of at most 16 tokens, or 32 if their activations fit (102400 x 2048, 32 tokens: 54 us, two
  // blocks of 16 60)
  const int most = t > MAX_COLS && fits(a.units.d, 2 * MAX_COLS) ? 2 * MAX_COLS : MAX_COLS;
  const int64_t blocks = ((int64_t)t + most - 1) / most;
  a.tb = (int)((t + blocks - 1) / blocks);
  const bool xr = a.x_vec && w->k % 8 == 0 && !fits(a.units.d, a.tb);
  if (!xr)
    while (a.tb > 1 && !fits(a.units.d, a.tb)) --a.tb;
  if (!xr && !fits(a.units.d, a.tb)) return fail(MK_EINVAL, "rows that are not 16-byte aligned are too long for the shared memory");
  a.cols = a.tb;
  a.ldr = ldr;
  a.ldo = ldo;
  a.out_f32 = out_f32;
  a.pairs = !out_f32 && aligned4(out, ldo) && (!residual || aligned4(residual, ldr));
  // a launch counts units of all its items in 32 bits: as many blocks at a time
  const int64_t most_items = INT32_MAX / 2 / ((int64_t)(w->n / 16 + 2) * a.units.d);
  if (!most_items) return fail(MK_EINVAL, "the weight is too large");
  for (int64_t at = 0; at < t; at += a.t) {
    a.t = (int)std::min(t - at, most_items * a.tb);
    a.n_items = (int)(((int64_t)a.t + a.tb - 1) / a.tb);
    a.x = static_cast<const uint16_t*>(x) + at * ldx;
    a.residual = residual ? static_cast<const uint16_t*>(residual) + at * ldr : nullptr;
    a.out = static_cast<uint8_t*>(out) + at * ldo * (out_f32 ? 4 : 2);
    if (int rc = launch_weight(a, w, a.n_items, true, xr, sms, static_cast<cudaStream_t>(stream))) return rc;
  }
  return MK_OK;
}

extern "C" int mk_w4_experts_workspace(const MkW4* w13, const MkW4* w2, int32_t t, int32_t slots, int64_t* bytes) {
  Plan p{};
  if (const char* m = plan_experts(w13, w2, t, slots, &p)) return fail(MK_EINVAL, m);
  if (!bytes) return fail(MK_EINVAL, "null pointer");
  *bytes = p.bytes;
  return MK_OK;
}

extern "C" int mk_w4_experts(const MkW4* w13, const MkW4* w2, const void* x, int64_t ldx, const int32_t* ids,
                             const float* weights, int32_t t, int32_t slots, const void* residual, int64_t ldr, void* out,
                             int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan p{};
  if (const char* m = plan_experts(w13, w2, t, slots, &p)) return fail(MK_EINVAL, m);
  if (t == 0) return MK_OK;
  if (!x || !out || (slots && (!ids || !weights))) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)x & 1) || ((uintptr_t)residual & 1) || ((uintptr_t)out & 1)) return fail(MK_EINVAL, "misaligned x, residual or out");
  if (((uintptr_t)ids & 3) || ((uintptr_t)weights & 3)) return fail(MK_EINVAL, "misaligned ids or weights");
  if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255))
    return fail(MK_EINVAL, "the workspace is missing, too small (mk_w4_experts_workspace) or not at a 256-byte boundary");
  int sms = 0;
  Args a{}, b{};
  if (int rc = device_sms(&a.device, &sms)) return rc;
  b.device = a.device;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t items_about = std::min<int64_t>((int64_t)t * slots, w13->experts);
  fill(a, w13);
  fill(b, w2);
  a.t = b.t = t;
  a.s = b.s = slots;
  a.s_div = b.s_div = div_by(std::max(slots, 1));
  a.ids = b.ids = ids;
  a.cols = b.cols = p.cols;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  a.out = ws + p.act;
  b.x = reinterpret_cast<const uint16_t*>(ws + p.act);
  b.x_vec = 1;
  if (p.small) {
    a.mode = GATEUP_SMALL;
    a.ldo = b.units.d;
    if (slots)
      if (int rc = launch_weight(a, w13, items_about, false, false, sms, st)) return rc;
    b.mode = DOWN_SMALL;
    b.follows = slots > 0;
    b.weights = weights;
    b.residual = static_cast<const uint16_t*>(residual);
    b.ldr = ldr;
    b.out = out;
    b.ldo = ldo;
    b.pairs = aligned4(out, ldo) && (!residual || aligned4(residual, ldr));
    return launch_weight(b, w2, 1, true, p.xr2, sms, st);
  }
  int4* items = reinterpret_cast<int4*>(ws + p.items);
  int* items_n = reinterpret_cast<int*>(ws + p.items_n);
  int* col_token = reinterpret_cast<int*>(ws + p.col_token);
  int* slot_col = reinterpret_cast<int*>(ws + p.slot_col);
  // the launches after it take counts and indices from its output: none without it
  const int n = t * slots, warps = std::min({32, PLAN_COUNTS / w13->experts, (n + 31) / 32});
  const int chunk = warps ? ((n + warps - 1) / warps + 31) / 32 * 32 : 0;
  cudaError_t e = launch_behind(plan_kernel, dim3(1), 1024, warps * w13->experts * 4, st, false, ids, n, (int)slots, (int)w13->experts,
                                p.cols, warps, chunk, items, items_n, col_token, slot_col);
  if (e != cudaSuccess) return fail(MK_ECUDA, cudaGetErrorString(e));
  a.mode = GATEUP;
  a.follows = b.follows = 1;
  a.items = b.items = items;
  a.items_n = b.items_n = items_n;
  a.col_token = col_token;
  a.ldo = b.ldx = 2 * p.ldact;
  if (int rc = launch_weight(a, w13, items_about, false, false, sms, st)) return rc;
  b.mode = DOWN;
  b.out = ws + p.y;
  b.ldo = w2->n;
  b.out_f32 = 1;
  if (int rc = launch_weight(b, w2, items_about, false, p.xr2, sms, st)) return rc;
  const dim3 grid((unsigned)t, (unsigned)((w2->n + 255) / 256));
  const float* y = reinterpret_cast<const float*>(ws + p.y);
  e = launch_behind(
      w2->dtype == MK_W4_BF16 ? combine_kernel<Bf16> : combine_kernel<Fp16>, grid, 256, 0, st, true, y, (const int*)slot_col, weights, (int)slots,
      (int)w2->n, static_cast<const uint16_t*>(residual), ldr, static_cast<uint16_t*>(out), ldo);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}
