// A decode step of the module over paged 4-bit caches as one library call: the sequence of launches
// that NSAAttention makes for a token, with nothing of the host between them (the calls of their own
// took 250 us of it, whatever the batch).
#include <stdio.h>

#include "../../include/nsa_hip.h"
#include "nsa_device.h"
#include "nsa_kernels.h"

namespace nsa {

// The blocks that a step completes, one request or another nearly every step of a ragged batch: eight
// launches over the closing requests alone, bound by their latency.  16 sequences of 8000 tokens (H32
// G2 dk 128), a block a step: the step 103 us (72 without one), 391 with the layers over all
// sequences by torch calls between the phases; 32 of 4000 at H64 G4 dk 192: 147 (113), 424.
//
// A token of a closing request a workgroup (i l + u: token u of the i-th such request's last l): its key of
// the ring to k [.][l][nk], in 16-byte pieces; and fresh[z] = whether z closes a block.
__device__ __forceinline__ int paged_closing(uint64_t closing, int i) {  // the i-th of them
  for (int j = 0; j < i; ++j) closing &= closing - 1;
  return __builtin_ctzll(closing);
}
__global__ void paged_gather_kernel(const uint4* tail, const int* token_lengths, uint64_t closing, int l, int Z, int nk, int nv,
                                    uint4* k, int* fresh) {
  const int row = blockIdx.x, i = row / l, u = row - i * l;
  const int z = paged_closing(closing, i), place = (max(token_lengths[z], 0) % l + u) % l;
  const uint4* src = tail + ((int64_t)z * l + place) * (nk + nv);
  for (int j = threadIdx.x; j < nk; j += blockDim.x) k[(int64_t)row * nk + j] = src[j];
  if (row == 0 && (int)threadIdx.x < Z) fresh[threadIdx.x] = (int)(closing >> threadIdx.x & 1);
}

// Block i of group g, a workgroup: R = mean_u relu(Y_u + C_u) and V_cmp = mean_u v_u (from the ring), a thread
// a 16-byte piece, the sums in the order of nsa_compress_fwd's.  Bound by latency: sixteen tokens' rows
// are on their way at once (all blocks of a step are few workgroups; nsa_compress_fwd's pooling, made
// for many, takes 16.5 us for two blocks of four groups at dk 192, this 8.8; with 32 rows 9.8).
template <typename T>
__global__ __launch_bounds__(256) void paged_pool_kernel(const uint4* Y, const uint4* C, const uint4* tail, const int* token_lengths,
                                                         uint64_t closing, int l, int nk, int nv, uint4* R, uint4* Vc) {
  constexpr int EPF = 16 / sizeof(typename Store<T>::type), U = 16;
  const int i = blockIdx.x, g = blockIdx.y, G = gridDim.y, nw = 2 * nk, pc = threadIdx.x;  // pieces of a key, of a value
  if (pc >= nw + nv) return;
  const int z = paged_closing(closing, i), start = max(token_lengths[z], 0) % l;
  const bool isv = pc >= nw;
  float acc[EPF];
#pragma unroll
  for (int k = 0; k < EPF; ++k) acc[k] = 0.f;
  // (no load of either kind under a condition of its lane: all of them are on their way at once)
  const uint4* rows = isv ? tail + (int64_t)z * l * G * (nk + nv) + G * nk + g * nv + pc - nw
                          : Y + ((int64_t)i * l * G + g) * nw + pc;
  const int pitch = G * (isv ? nk + nv : nw), turn = isv ? start : 0;
  const uint4* bias = C + (isv ? 0 : pc);
  for (int u0 = 0; u0 < l; u0 += U) {
    uint4 x[U], c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(u0 + u, l - 1), place = turn + t < l ? turn + t : turn + t - l;
      x[u] = rows[(int64_t)place * pitch];
      c[u] = bias[t * nw];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[EPF], b[EPF];
      unpack16<T>(x[u], y);
      unpack16<T>(c[u], b);
#pragma unroll
      for (int k = 0; k < EPF; ++k) {
        const float s = isv ? y[k] : y[k] + b[k], v = isv || s > 0.f ? s : 0.f;
        acc[k] = u0 + u < l ? acc[k] + v : acc[k];
      }
    }
  }
  const float inv = 1.0f / (float)l;
#pragma unroll
  for (int k = 0; k < EPF; ++k) acc[k] *= inv;
  const int64_t row = (int64_t)i * G + g;
  if (isv) Vc[row * nv + pc - nw] = pack16<T>(acc);
  else R[row * nw + pc] = pack16<T>(acc);
}

// The i-th new block's key of group g, a workgroup, to its place among the request's.
__global__ void paged_keys_kernel(const uint4* k, int pieces, const int* sequences, const int* positions, uint4* k_cmp,
                                  int64_t kz, int64_t kg, int64_t kn) {
  const int i = blockIdx.x, g = blockIdx.y, z = sequences[i], at = positions[i];
  if (z < 0 || at < 0) return;
  for (int j = threadIdx.x; j < pieces; j += blockDim.x)
    k_cmp[z * kz + g * kg + at * kn + j] = k[((int64_t)i * gridDim.y + g) * pieces + j];
}

struct PagedBlocksLayout {
  size_t k, y, c, r, kc, vc, fresh, slots, positions, sequences, total;
  int n;
};

static int paged_blocks_shape(const nsa_paged_blocks_args& x, PagedBlocksLayout& L) {
  if (x.dtype != NSA_F32 && x.dtype != NSA_BF16) return set_error(NSA_ERR_INVALID, "dtype not supported");
  if (x.Z < 1 || x.Z > 64 || x.n_kv_groups < 1 || x.n_kv_groups > 65535 || !x.closing || (x.Z < 64 && x.closing >> x.Z))
    return set_error(NSA_ERR_INVALID, "bad shape, or closing names no request");
  const int64_t es = x.dtype == NSA_F32 ? 4 : 2, epf = 16 / es, G = x.n_kv_groups, dk = x.head_dim_qk, dv = x.head_dim_v;
  if (x.l < 1 || x.l > 64 || x.l % epf || dk <= 0 || dk % 64 || dv <= 0 || dv % epf || (2 * dk + dv) / epf > 256 ||
      !nsa_head_dims_supported(x.dtype, x.head_dim_qk, x.head_dim_v))
    return set_error(NSA_ERR_UNSUPPORTED, "paged blocks: widths without a kernel");
  L.n = __builtin_popcountll(x.closing);
  size_t off = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = off;
    off += ((size_t)bytes + 255) & ~(size_t)255;
    return o;
  };
  L.k = take(L.n * x.l * G * dk * es);
  L.y = take(L.n * x.l * G * 2 * dk * es);
  L.c = take(x.l * 2 * dk * es);
  L.r = take(L.n * G * 2 * dk * es);
  L.kc = take(L.n * G * dk * es);
  L.vc = take(L.n * G * dv * es);
  L.fresh = take(x.Z * 4);
  L.slots = take(L.n * 8);
  L.positions = take(L.n * 4);
  L.sequences = take(L.n * 4);
  L.total = off;
  return NSA_OK;
}

static int paged_blocks_check(const nsa_paged_blocks_args& x, PagedBlocksLayout& L) {
  const int rc = paged_blocks_shape(x, L);
  if (rc) return rc;
  const void* need[] = {x.pages, x.tables, x.token_lengths, x.lengths, x.free_pages, x.used, x.state, x.tail, x.k_cmp, x.E,
                        x.W1, x.W2};
  for (const void* p : need)
    if (!p) return set_error(NSA_ERR_INVALID, "paged blocks: null tensor");
  const int epf = x.dtype == NSA_F32 ? 4 : 8;
  if (((uintptr_t)x.tail | (uintptr_t)x.k_cmp | (uintptr_t)x.E | (uintptr_t)x.W1 | (uintptr_t)x.W2) % 16 ||
      x.stride_kz % epf || x.stride_kg % epf || x.stride_kn % epf)
    return set_error(NSA_ERR_LAYOUT, "paged blocks: tensors need 16-byte aligned rows");
  return NSA_OK;
}

static int paged_blocks(const nsa_paged_blocks_args& x, const PagedBlocksLayout& L, char* base, nsa_stream_t stream) {
  const int es = x.dtype == NSA_F32 ? 4 : 2, G = x.n_kv_groups, dk = x.head_dim_qk, dv = x.head_dim_v, W = 2 * dk, l = x.l;
  const int epf = 16 / es;
  hipStream_t st = (hipStream_t)stream;
  auto vec = [&](size_t o) { return reinterpret_cast<uint4*>(base + o); };
  auto ints = [&](size_t o) { return reinterpret_cast<int*>(base + o); };
  hipLaunchKernelGGL(paged_gather_kernel, dim3(L.n * l), dim3(64), 0, st, static_cast<const uint4*>(x.tail), x.token_lengths,
                     x.closing, l, x.Z, G * dk / epf, G * dv / epf, vec(L.k), ints(L.fresh));
  // Y = k W1[:, :dk]^T, C = E W1[:, dk:]^T + b1, the pooling, K = R W2^T + b2
  int rc;
  const nsa_linear_job y{x.W1, nullptr, base + L.y, dk + l, W, 0, W, W, 0};
  if ((rc = launch_linear_rows(base + L.k, dk, L.n * l * G, dk, 1, 0, 0, y, x.dtype, st))) return rc;
  const nsa_linear_job c{static_cast<const char*>(x.W1) + (int64_t)dk * es, x.b1, base + L.c, dk + l, W, 0, W, W, 0};
  if ((rc = launch_linear_rows(x.E, l, l, l, 1, 0, 0, c, x.dtype, st))) return rc;
  auto pool = x.dtype == NSA_F32 ? paged_pool_kernel<float> : paged_pool_kernel<bf16>;
  hipLaunchKernelGGL(pool, dim3(L.n, G), dim3(256), 0, st, vec(L.y), vec(L.c), static_cast<const uint4*>(x.tail), x.token_lengths,
                     x.closing, l, dk / epf, dv / epf, vec(L.r), vec(L.vc));
  const nsa_linear_job k{x.W2, x.b2, base + L.kc, W, dk, 0, dk, dk, 0};
  if ((rc = launch_linear_rows(base + L.r, W, L.n * G, W, 1, 0, 0, k, x.dtype, st))) return rc;
  int64_t* slots = reinterpret_cast<int64_t*>(base + L.slots);
  rc = nsa_block_tables(x.tables, x.stride_table, x.Z, x.table_width, x.lengths, ints(L.fresh), x.free_pages, x.n_free, x.used,
                        x.pages->page_size, L.n, 0, slots, ints(L.positions), ints(L.sequences), x.state, x.state + x.Z + 1,
                        x.state + 2 * x.Z + 1, stream);
  if (rc) return rc;
  rc = nsa_kv4_store(x.pages, base + L.kc, (int64_t)G * dk, dk, base + L.vc, (int64_t)G * dv, dv, slots, L.n, G, dk, dv, x.dtype,
                     stream);
  if (rc) return rc;
  hipLaunchKernelGGL(paged_keys_kernel, dim3(L.n, G), dim3(64), 0, st, vec(L.kc), dk / epf, ints(L.sequences),
                     ints(L.positions), static_cast<uint4*>(x.k_cmp), x.stride_kz / epf, x.stride_kg / epf, x.stride_kn / epf);
  return hipGetLastError() == hipSuccess ? NSA_OK : set_error(NSA_ERR_HIP, "paged blocks launch failed");
}

// Offsets of the workspace.
struct PagedStepLayout {
  size_t q, hid, z, o, idx, rows, slots, positions, sequences, seen, score, attn, blocks, total, score_bytes, attn_bytes;
  PagedBlocksLayout closing;
};

static nsa_kv4_attn_args paged_step_attn(const nsa_paged_step_args& x) {
  nsa_kv4_attn_args a{};
  for (int s = 0; s < 3; ++s) {
    a.pages[s] = x.pages[s];
    a.tables[s] = s == 0 ? x.cmp_tables : x.tables;
    a.stride_table[s] = s == 0 ? x.stride_cmp_table : x.stride_table;
    a.table_width[s] = s == 0 ? x.cmp_table_width : x.table_width;
  }
  const int64_t H = x.H, dk = x.head_dim_qk, dv = x.head_dim_v;
  a.stride_qz = a.stride_qt = H * dk, a.stride_qh = dk;
  a.stride_oz = a.stride_ot = H * dv, a.stride_oh = dv;
  a.stride_gz = a.stride_gt = 3 * H, a.stride_gh = 3, a.stride_gk = 1;
  a.Z = x.Z, a.H = x.H, a.n_kv_groups = x.n_kv_groups, a.n_ctx_q = 1;
  a.head_dim_qk = x.head_dim_qk, a.head_dim_v = x.head_dim_v, a.max_length = x.max_length;
  a.l = x.l, a.d = x.d, a.n_slots = x.n, a.block_size_selection = x.l_prime, a.window_size = x.window_size;
  a.gate_act = x.gate_act, a.dtype = x.dtype, a.sm_scale = x.sm_scale;
  a.gates = &x;  // (there are some: their address comes with the workspace)
  return a;
}

// The step's sizes checked; its layout and attention arguments.
static int paged_step_shape(const nsa_paged_step_args& x, nsa_kv4_attn_args& a, PagedStepLayout& L) {
  if (x.dtype != NSA_F32 && x.dtype != NSA_BF16) return set_error(NSA_ERR_INVALID, "dtype not supported");
  if (x.Z < 1 || x.Z > 64 || x.H < 1 || x.n_kv_groups < 1 || x.H % x.n_kv_groups || x.d_model < 1 || x.gate_hidden < 1 ||
      x.n_blocks < 1 || x.l < 1 || x.d < 1 || x.n < 1)
    return set_error(NSA_ERR_INVALID, "bad shape");
  if (!nsa_head_dims_supported(x.dtype, x.head_dim_qk, x.head_dim_v))
    return set_error(NSA_ERR_UNSUPPORTED, "no kernel for these head dims");
  if (!x.pages[0] || !x.pages[1] || !x.pages[2] || x.pages[1]->page_size != x.pages[2]->page_size)
    return set_error(NSA_ERR_INVALID, "null pages, or selection and window of different page sizes");
  a = paged_step_attn(x);
  L = PagedStepLayout{};
  L.attn_bytes = nsa_kv4_attn_workspace_size(&a);
  L.score_bytes = nsa_score_topn_workspace_size(x.Z, x.H, x.n_kv_groups, 1, x.head_dim_qk, x.n_blocks, x.n);
  const size_t es = x.dtype == NSA_F32 ? 4 : 2, Z = x.Z, H = x.H, G = x.n_kv_groups;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off += (bytes + 255) & ~(size_t)255;
    return o;
  };
  L.q = take(Z * H * x.head_dim_qk * es);
  L.hid = take(Z * x.gate_hidden * es);
  L.z = take(Z * H * 3 * es);
  L.o = take(Z * H * x.head_dim_v * es);
  L.idx = take(Z * G * x.n * 8);
  L.rows = take(Z * 3 * G * (x.head_dim_qk + x.head_dim_v) * es);
  L.slots = take(Z * 8);
  L.positions = take(Z * 4);
  L.sequences = take(Z * 4);
  L.seen = take(Z * 4);
  L.score = take(L.score_bytes);
  L.attn = take(L.attn_bytes);
  if (x.blocks) {
    if (const int rc = paged_blocks_shape(*x.blocks, L.closing)) return rc;
    L.blocks = take(L.closing.total);
  }
  L.total = off;
  return NSA_OK;
}

}  // namespace nsa

using namespace nsa;

extern "C" size_t nsa_paged_blocks_workspace_size(const nsa_paged_blocks_args* x) {
  PagedBlocksLayout L;
  return !x || paged_blocks_shape(*x, L) ? 0 : L.total;
}

extern "C" int nsa_paged_blocks(const nsa_paged_blocks_args* x, void* ws, size_t ws_bytes, nsa_stream_t stream) {
  if (!x) return set_error(NSA_ERR_INVALID, "args is null");
  PagedBlocksLayout L;
  const int rc = paged_blocks_check(*x, L);
  if (rc) return rc;
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < L.total) {
    char msg[128];
    snprintf(msg, sizeof(msg), "workspace of %zu bytes (16-byte aligned) required, %zu given", L.total, ws_bytes);
    return set_error(NSA_ERR_WORKSPACE, msg);
  }
  return paged_blocks(*x, L, static_cast<char*>(ws), stream);
}

extern "C" size_t nsa_paged_step_workspace_size(const nsa_paged_step_args* x) {
  nsa_kv4_attn_args a;
  PagedStepLayout L;
  return !x || paged_step_shape(*x, a, L) ? 0 : L.total;
}

extern "C" int nsa_paged_step(const nsa_paged_step_args* x, void* ws, size_t ws_bytes, nsa_stream_t stream) {
  if (!x) return set_error(NSA_ERR_INVALID, "args is null");
  nsa_kv4_attn_args a;
  PagedStepLayout L;
  int rc = paged_step_shape(*x, a, L);
  if (rc) return rc;
  if (!(x->phases & 3) || (x->phases & ~3)) return set_error(NSA_ERR_INVALID, "phases outside [1, 3]");
  if (!x->tables || !x->cmp_tables || !x->lengths || !x->new_tokens || !x->free_pages || !x->used || !x->state || !x->tail ||
      !x->k_cmp || !x->block_ends || !x->out || !x->x)
    return set_error(NSA_ERR_INVALID, "null tensor");
  if ((uintptr_t)x->tail % 16) return set_error(NSA_ERR_LAYOUT, "tail must be 16-byte aligned");
  if (x->blocks && (rc = paged_blocks_check(*x->blocks, L.closing))) return rc;
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < L.total) {
    char msg[128];
    snprintf(msg, sizeof(msg), "workspace of %zu bytes (16-byte aligned) required, %zu given", L.total, ws_bytes);
    return set_error(NSA_ERR_WORKSPACE, msg);
  }
  char* base = static_cast<char*>(ws);
  const int Z = x->Z, H = x->H, G = x->n_kv_groups, dk = x->head_dim_qk, dv = x->head_dim_v, hw = x->gate_hidden;
  const int es = x->dtype == NSA_F32 ? 4 : 2;
  const int64_t ld = (int64_t)3 * G * (dk + dv);
  void *q = base + L.q, *hid = base + L.hid, *z = base + L.z, *o = base + L.o;
  int *positions = reinterpret_cast<int*>(base + L.positions), *seen = reinterpret_cast<int*>(base + L.seen);
  auto job = [&](int i, void* out, int n, int64_t row, int relu) {
    return nsa_linear_job{x->w[i], x->bias[i], out, x->ldw[i], row, 0, n, n, relu};
  };
  if (x->phases & 1) {
    Kv4Pages sel, win;
    if ((rc = kv4_check_pages(x->pages[1], G, &sel)) || (rc = kv4_check_pages(x->pages[2], G, &win))) return rc;
    nsa_linear_job jobs[8];
    jobs[0] = job(0, q, H * dk, (int64_t)H * dk, 0);
    jobs[1] = job(7, hid, hw, hw, 1);
    int64_t at = 0;
    for (int i = 0; i < 6; ++i) {
      const int n = G * (i & 1 ? dv : dk);
      jobs[2 + i] = job(1 + i, base + L.rows + at * es, n, ld, 0);
      at += n;
    }
    if ((rc = nsa_linear_few(x->x, x->ld_x, Z, x->d_model, jobs, 8, x->dtype, stream))) return rc;
    const nsa_linear_job gate = job(8, z, 3 * H, 3 * H, 0);
    if ((rc = nsa_linear_few(hid, hw, Z, hw, &gate, 1, x->dtype, stream))) return rc;
    int64_t* slots = reinterpret_cast<int64_t*>(base + L.slots);
    rc = nsa_block_tables(x->tables, x->stride_table, Z, x->table_width, x->lengths, x->new_tokens, x->free_pages, x->n_free,
                          x->used, x->pages[1]->page_size, Z, 1, slots, positions, reinterpret_cast<int*>(base + L.sequences),
                          x->state, x->state + Z + 1, x->state + 2 * Z + 1, stream);
    if (rc) return rc;
    const PagedTail tail{static_cast<uint4*>(x->tail), x->lengths, positions, seen, Z, x->l, nullptr, 0, 0};
    if ((rc = launch_paged_put(x->dtype, dk, dv, G, base + L.rows, ld, sel, win, slots, tail, (hipStream_t)stream))) return rc;
  }
  if (x->blocks && (rc = paged_blocks(*x->blocks, L.closing, base + L.blocks, stream))) return rc;
  if (x->phases & 2) {
    int64_t* idx = reinterpret_cast<int64_t*>(base + L.idx);
    rc = nsa_score_topn_at(q, x->k_cmp, x->block_ends, idx, nullptr, nullptr, (int64_t)H * dk, dk, dk, 1, x->stride_kz,
                           x->stride_kg, 1, x->stride_kn, (int64_t)G * x->n, x->n, x->n, 1, Z, H, G, 1, dk, x->n_blocks, x->l,
                           x->d, x->l_prime, x->n, x->include_fixed, x->n_fixed, x->dtype, x->sm_scale, positions,
                           base + L.score, L.score_bytes, stream);
    if (rc) return rc;
    a.q = q;
    a.gates = z;
    a.indices = idx;
    a.lengths = seen;
    a.out = o;
    if (!x->w[9]) {  // no output projection: the mixed heads are the result
      a.out = x->out;
      a.stride_oz = a.stride_ot = x->ld_out;
    }
    if ((rc = nsa_kv4_attn(&a, base + L.attn, L.attn_bytes, stream))) return rc;
    if (!x->w[9]) return NSA_OK;
    const nsa_linear_job out = job(9, x->out, x->d_model, x->ld_out, 0);
    if ((rc = nsa_linear_few(o, (int64_t)H * dv, Z, H * dv, &out, 1, x->dtype, stream))) return rc;
  }
  return NSA_OK;
}
