// lx_linear_attention: linear attention with a decay for each head, a state of each sequence and head kept between calls.
#include "linear_chunk.h"
#include "linear_step.h"

namespace dro {
namespace {

constexpr int kMaxDk = 256, kMaxDv = 512, kMaxHeads = 4096;
constexpr int kMaxStride = 1 << 22;  // values: rows of a chunk are told apart in 31 bits
// Rows of a sequence that go token by token; from there on by chunks, whose products cost the same for one row and 64. The two cross at 5 rows where the states of some sequences
// fill the device, at 9 where one does not or where many are bound by their bytes: one number between them, so that a token's roundings go by max_rows alone. By tokens and by a
// chunk, 128 heads of 128 by 64: 8 sequences of 4 rows 17.4 us and 19.6, of 6 21.0 and 19.7, of 8 24.5 and 19.8, of 16 38.5 and 20.8; 64 sequences of 4 103 and 140, of 8 138 and
// 145, of 12 175 and 148; one sequence of 32 heads of 128 by 128, 4 rows 7.2 and 11.6, 8 rows 10.3 and 11.6, 12 rows 13.5 and 11.6.
constexpr int kMostSteps = 6;

template <int COLS, int ROWS>
int launch_step(const LinearArgs& p, hipStream_t s) {
  const int64_t waves = static_cast<int64_t>(p.b.seqs) * p.heads * ((p.dv + 4 * COLS - 1) / (4 * COLS));
  const int64_t groups = (waves + 3) / 4;
  if (groups * 256 > kMaxGridThreads) return kInvalid;
  const auto kernel = p.type == LX_BF16 && p.wide && (!p.gate || p.gate_type == LX_BF16) ? linear_step_kernel<COLS, ROWS, true> : linear_step_kernel<COLS, ROWS, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, p);
  return status_of(hipGetLastError());
}

int steps(const LinearArgs& p, hipStream_t s) {
  if (p.dk <= 64) return launch_step<8, 8>(p, s);
  // 16 columns a wavefront where 32 leave the device short of wavefronts (sums are made in the same order): one sequence of 32 heads of 128 by 128 4.0 us, 4.6 by 32; eight of 128
  // heads of 128 by 64, 2048 wavefronts of 32 columns, 17.6 us and 18.1 by 16.
  const bool few = static_cast<int64_t>(p.b.seqs) * p.heads * ((p.dv + 31) / 32) < 4 * compute_units();
  if (p.dk <= 128) return few ? launch_step<4, 8>(p, s) : launch_step<8, 16>(p, s);
  return few ? launch_step<4, 16>(p, s) : launch_step<8, 32>(p, s);
}

// How a call of chunks is cut: heads (or columns of wide ones) by workgroups, long sequences into parts of `size` rows.
struct Cut {
  int waves, teams;  // of a head's columns, heads of a workgroup
  int across;        // workgroups of a key head
  int size, places;  // rows of a part; parts of long sequences there may be
};

constexpr int kLeastPart = 128;  // rows; five sequences of up to 611 rows of 12 heads 33.8 us, 43.9 by 256
// Of sequences of so many parts the outputs' kernel adds up what is in front of a part by itself; of more, where that would be most of what it reads, a kernel in between
// runs through them once. 4096 tokens of 128 heads, 8 parts: 128 us and 138; eight sequences of up to 4 parts of 8 heads of 256 by 256: 126 and 161.
constexpr int kFewParts = 8;

Cut cut_of(int T, int max_rows, int heads, int k_heads, int dk, int dv) {
  Cut c;
  const int group = heads / k_heads;
  // A head of 64 columns or fewer has two wavefronts, and a workgroup two such heads, if there are two that read the same keys (4096 tokens of 128 heads, 16 of
  // them to a key head: 128 us, 173 by one head a workgroup); 256 keys' values are too many loads for two wavefronts.
  c.teams = dv <= 64 && group > 1 ? 2 : 1;
  c.waves = dv <= 64 && (c.teams == 2 || dk <= 128) ? 2 : 4;
  c.across = c.teams > 1 ? (group + 1) / 2 : group * ((dv + 32 * c.waves - 1) / (32 * c.waves));
  // As many parts as two workgroups a unit of the device: a part costs a second look at its keys and values, but few of them end together. By one, two and four
  // workgroups a unit: 4096 tokens of 128 heads 161, 128 and 173 us, 16384 of 16 heads 145, 134 and 168 us; eight prompts of up to 2048 of 8 heads of 256 by 256, of which
  // a unit has one at a time, 135, 126 and 235 us.
  const int64_t places = 2 * static_cast<int64_t>(compute_units()), columns = static_cast<int64_t>(c.across) * k_heads;
  const int64_t even = (T * columns + places - 1) / places, size = (even + kChunk - 1) / kChunk * kChunk;
  c.size = static_cast<int>(size < kLeastPart ? kLeastPart : size);
  // No call of T rows or fewer has more: a part is no shorter than T columns / places.
  const int64_t most = T / kLeastPart < places / columns ? T / kLeastPart : places / columns;
  c.places = static_cast<int>(2 * most);
  if (max_rows <= c.size) c.size = (max_rows + kChunk - 1) / kChunk * kChunk;
  return c;
}

int64_t sum_bytes(const Cut& c, int heads, int dk, int dv) { return 4 * static_cast<int64_t>(c.places) * heads * part_values(dk, dv); }

template <int DK, int TW, int TEAMS, bool OUT, bool PLAIN, int TERMS>
int launch_kernel(const ChunkArgs& a, int64_t groups, hipStream_t s) {
  constexpr int kHalves = DK > 128 ? 2 : 1;
  using L = ChunkTiles<DK, TW, TEAMS, kHalves, TERMS>;
  constexpr int kLds = OUT ? L::kBytes : L::kSumBytes;
  if (groups * L::kThreads > kMaxGridThreads) return kInvalid;
  const auto kernel = linear_chunk_kernel<DK, TW, TEAMS, kHalves, OUT, PLAIN, TERMS>;
  allow_lds(reinterpret_cast<const void*>(kernel), kLds);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(L::kThreads), kLds, s, a);
  return status_of(hipGetLastError());
}

template <int DK, int TW, int TEAMS, bool OUT>
int launch_chunks(ChunkArgs a, int64_t numbers, hipStream_t s) {
  a.numbers = numbers;
  const int64_t groups = (numbers * a.l.k_heads + 7) / 8 * 8 * a.across;
  const bool plain = a.l.type == LX_BF16 && a.l.wide && (!a.l.gate || a.l.gate_type == LX_BF16);
  if constexpr (OUT) {
    if (plain && a.l.out_type == LX_BF16) return launch_kernel<DK, TW, TEAMS, true, true, 2>(a, groups, s);
    return plain ? launch_kernel<DK, TW, TEAMS, true, true, 3>(a, groups, s) : launch_kernel<DK, TW, TEAMS, true, false, 3>(a, groups, s);
  } else {
    return plain ? launch_kernel<DK, TW, TEAMS, false, true, 2>(a, groups, s) : launch_kernel<DK, TW, TEAMS, false, false, 2>(a, groups, s);
  }
}

template <int DK, int TW, int TEAMS>
int chunks_of(const ChunkArgs& a, hipStream_t s) {
  const MixBatch& b = a.l.b;
  if (!a.single) {
    const int64_t places = 2 * static_cast<int64_t>(b.T / a.size);
    if (int st = launch_chunks<DK, TW, TEAMS, false>(a, places, s)) return st;
    if (!a.sums_only) {
      const int64_t fours = a.l.heads * part_values(a.l.dk, a.l.dv) / 4, groups = (fours + 255) / 256 * (places / 2);
      if (groups * 256 > kMaxGridThreads) return kInvalid;
      hipLaunchKernelGGL(linear_parts_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, a);
      if (int st = status_of(hipGetLastError())) return st;
    }
  }
  return launch_chunks<DK, TW, TEAMS, true>(a, mix_piece_count(b, MixPieces{a.size, a.single}), s);
}

template <int DK>
int chunks_by(const ChunkArgs& a, const Cut& c, hipStream_t s) {
  if (c.waves == 4) return chunks_of<DK, 4, 1>(a, s);
  if (c.teams == 2) return chunks_of<DK, 2, 2>(a, s);
  if constexpr (DK <= 128) return chunks_of<DK, 2, 1>(a, s);
  return kInvalid;
}

int chunks(const LinearArgs& p, void* workspace, hipStream_t s) {
  const Cut c = cut_of(p.b.T, p.b.max_rows, p.heads, p.k_heads, p.dk, p.dv);
  ChunkArgs a{};
  a.l = p, a.size = c.size, a.single = mix_pieces(p.b, c.size).single, a.across = c.across;
  a.sums_only = p.b.max_rows <= kFewParts * c.size;
  if (!a.single) {
    if (!workspace) return kInvalid;
    a.sums = static_cast<float*>(workspace);
    a.logs = reinterpret_cast<double*>(static_cast<char*>(workspace) + sum_bytes(c, p.heads, p.dk, p.dv));
  }
  return p.dk <= 64 ? chunks_by<64>(a, c, s) : p.dk <= 128 ? chunks_by<128>(a, c, s) : chunks_by<256>(a, c, s);
}

bool sizes_known(int T, int heads, int k_heads, int dk, int dv) {
  return T >= 0 && T < (1 << 30) && k_heads >= 1 && heads >= k_heads && heads <= kMaxHeads && heads % k_heads == 0 && dk >= 8 && dk <= kMaxDk &&
         dk % 8 == 0 && dv >= 8 && dv <= kMaxDv && dv % 8 == 0;
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int64_t lx_linear_attention_workspace_bytes(const lx_kv8_batch* batch, int T, int heads, int k_heads, int dk, int dv) {
  if (!batch || !sizes_known(T, heads, k_heads, dk, dv)) return -1;
  const Cut c = cut_of(T, T, heads, k_heads, dk, dv);
  return sum_bytes(c, heads, dk, dv) + 8 * static_cast<int64_t>(c.places) * heads;
}

int lx_linear_attention(const void* q, const void* k, const void* v, lx_dtype dtype, int ld_q, int ld_k, int ld_v, const lx_decay* decay,
                        const float* skip, const void* gate, lx_dtype gate_dtype, int ld_gate, const lx_kv8_batch* batch,
                        const lx_states* states, void* out, lx_dtype out_dtype, int ld_out, int T, int heads, int k_heads, int dk, int dv,
                        float scale, void* workspace, void* stream) {
  if (!sizes_known(T, heads, k_heads, dk, dv)) return fail(kInvalid);
  if (int st = mix_check(batch, T)) return fail(st);
  if (int st = mix_check_states(states)) return fail(st);
  if (!mix_type(dtype) || !mix_type(out_dtype) || (gate && !mix_type(gate_dtype))) return fail(kInvalid);
  if (!decay || (decay->kind != LX_DECAY_HEAD && decay->kind != LX_DECAY_LOG && decay->kind != LX_DECAY_STEP)) return fail(kInvalid);
  if (states && (reinterpret_cast<uintptr_t>(states->in) | reinterpret_cast<uintptr_t>(states->out)) % 16 != 0) return fail(kInvalid);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(kInvalid);
  const bool by_token = decay->kind != LX_DECAY_HEAD;
  if (by_token && !mix_type(decay->dtype)) return fail(kInvalid);
  if (T == 0 || batch->seqs == 0) return kOk;
  if (!q || !k || !v || !out || (by_token ? !decay->x : !decay->rate)) return fail(kInvalid);
  const int64_t keys = static_cast<int64_t>(k_heads) * dk, values = static_cast<int64_t>(heads) * dv;
  if (T > 1 && (ld_q < keys || ld_k < keys || ld_v < values || ld_out < values || (gate && ld_gate < values) || (by_token && decay->ld < heads)))
    return fail(kInvalid);
  if (T > 1 && (ld_q > kMaxStride || ld_k > kMaxStride || ld_v > kMaxStride || ld_out > kMaxStride || (gate && ld_gate > kMaxStride))) return fail(kInvalid);
  LinearArgs p{};
  p.q = q, p.k = k, p.v = v, p.x = by_token ? decay->x : nullptr, p.rate = decay->rate;
  p.bias = decay->kind == LX_DECAY_STEP ? decay->bias : nullptr;
  p.skip = skip, p.gate = gate, p.out = out;
  p.ld_q = ld_q, p.ld_k = ld_k, p.ld_v = ld_v, p.ld_x = decay->ld, p.ld_gate = ld_gate, p.ld_out = ld_out;
  p.type = dtype, p.x_type = decay->dtype, p.gate_type = gate_dtype, p.out_type = out_dtype;
  p.kind = decay->kind, p.heads = heads, p.k_heads = k_heads, p.group = heads / k_heads, p.dk = dk, p.dv = dv;
  auto in16 = [&](const void* t, int ld, int type) { return mix_aligned(t, T > 1 ? ld : 0, type, 16); };
  p.wide = in16(q, ld_q, dtype) && in16(k, ld_k, dtype) && in16(v, ld_v, dtype) && (!gate || in16(gate, ld_gate, gate_dtype)) && in16(out, ld_out, out_dtype);
  p.scale = scale;
  p.b = mix_batch(*batch, T);
  p.states = mix_states(states);
  if (p.b.max_rows == 0 || p.b.seqs == 0) return kOk;
  // Other columns' workgroups still read what a result would replace.
  if (out == q || out == k || out == v || out == gate || out == p.x) return fail(kInvalid);
  const int st = p.b.max_rows <= kMostSteps ? steps(p, as_stream(stream)) : chunks(p, workspace, as_stream(stream));
  return st ? fail(st) : kOk;
}

}  // extern "C"
