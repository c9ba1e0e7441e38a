// C-ABI entry points that write rows into KV caches and read them back without
// attention (see include/qm38.h).
#include <math.h>

#include <algorithm>

#include "kv_append.h"
#include "kv_internal.h"

using namespace qm;

namespace {

KvPages pages_of(const qm_kv* kv) {
  return KvPages{(uint8_t*)kv->k, (uint8_t*)kv->v, kv->ks, kv->vs, kv->d_pt};
}

// Rows of a call: the append's index arithmetic and its launch stay within 32 bits.
constexpr uint64_t kMaxRows = 1u << 20;

}  // namespace

extern "C" {

qm_status qm_kv_append(qm_runtime* rt, qm_kv* const* seqs, const uint32_t* counts, uint32_t B, const qm_kv_rows* rows) {
  if (!rt || !seqs || !counts || !rows || !rows->k || !rows->v) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (B == 0 || B > 64) return fail(QM_ERR_INVALID_ARGUMENT, "batch must be 1..64 sequences");
  const qm_kv* s0 = seqs[0];
  if (!s0) return fail(QM_ERR_NULL_POINTER, "sequence 0 is NULL");
  const uint32_t KVH = s0->kv_heads, D = s0->head_dim;
  uint64_t total = 0, units = 0;
  for (uint32_t b = 0; b < B; ++b) {
    const qm_kv* kv = seqs[b];
    if (!kv) return fail(QM_ERR_NULL_POINTER, "sequence %u is NULL", b);
    if (kv->kv_heads != KVH || kv->head_dim != D)
      return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "all sequences must share kv_heads and head_dim");
    if (kv->bits != s0->bits) return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "8-bit and 4-bit caches in one call");
    if (kv->rt->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "sequence %u is on another device", b);
    for (uint32_t c = 0; c < b; ++c)
      if (seqs[c] == kv) return fail(QM_ERR_INVALID_ARGUMENT, "sequence %u appears twice", b);
    if ((uint64_t)kv->length + counts[b] > 0xFFFFFFFFull) return fail(QM_ERR_DIMENSION_OVERFLOW, "KV token capacity");
    total += counts[b];
    units += ((uint64_t)counts[b] / 16 + 2) * KVH;
  }
  if (total == 0) return fail(QM_ERR_EMPTY_APPEND, "no row to append");
  if (total > kMaxRows) return fail(QM_ERR_DIMENSION_OVERFLOW, "%llu rows in one call", (unsigned long long)total);

  KvAppendArgs a{};
  a.k = rows->k;
  a.v = rows->v;
  const uint64_t width = (uint64_t)KVH * D;
  a.k_stride = rows->k_stride ? rows->k_stride : width;
  a.v_stride = rows->v_stride ? rows->v_stride : width;
  if (a.k_stride < width || a.v_stride < width)
    return fail(QM_ERR_INVALID_ARGUMENT, "a row stride is below kv_heads * head_dim = %llu", (unsigned long long)width);
  if (std::max(a.k_stride, a.v_stride) > (1ull << 62) / total) return fail(QM_ERR_DIMENSION_OVERFLOW, "rows * stride");
  if (!aligned(rows->k, 2) || !aligned(rows->v, 2)) return fail(QM_ERR_MISALIGNED, "k and v need 2-byte alignment");
  if (!aligned(rows->positions, 4)) return fail(QM_ERR_MISALIGNED, "positions must be 4-byte aligned");
  bool vec = D % 4 == 0 && aligned(a.k, 8) && aligned(a.v, 8) && (total == 1 || (a.k_stride % 4 == 0 && a.v_stride % 4 == 0));
  bool interleaved = false, qvec = false;
  if (rows->rotary) {
    qm_status st = rotary_frequencies(*rows->rotary, a.freq, &a.factor);
    if (st != QM_OK) return st;
    const uint32_t rd = rows->rotary->rotary_dim;
    if ((uint64_t)rows->offset + rd > D)
      return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "elements %u .. %u + %u pass head_dim %u", rows->offset, rows->offset, rd, D);
    interleaved = rows->rotary->layout == QM_ROTARY_INTERLEAVED;
    a.rotary_dim = rd;
    a.offset = rows->offset;
    a.positions = rows->positions;
    vec = vec && rows->offset % 4 == 0 && rd % (interleaved ? 4 : 8) == 0;
  }
  if (rows->q) {
    if (!rows->rotary) return fail(QM_ERR_INVALID_ARGUMENT, "queries are only rotated: no rotary configuration");
    if (!rows->q_out) return fail(QM_ERR_NULL_POINTER, "q_out is NULL");
    if (rows->heads == 0) return fail(QM_ERR_EMPTY_DIMENSION, "heads must be > 0");
    RotaryTensor& t = a.q;
    const uint64_t qwidth = (uint64_t)rows->heads * D;
    if (qwidth > 0x7FFFFFFFull) return fail(QM_ERR_DIMENSION_OVERFLOW, "a row of queries passes 2^31 - 1 elements");
    t.in = rows->q;
    t.out = rows->q_out;
    t.in_stride = rows->q_stride ? rows->q_stride : qwidth;
    t.out_stride = rows->q_out_stride ? rows->q_out_stride : qwidth;
    t.heads = rows->heads;
    t.head_dim = D;
    t.offset = rows->offset;
    if (t.in_stride < qwidth || t.out_stride < qwidth)
      return fail(QM_ERR_INVALID_ARGUMENT, "a row stride of the queries is below heads * head_dim = %llu",
                  (unsigned long long)qwidth);
    if (std::max(t.in_stride, t.out_stride) > (1ull << 62) / total)
      return fail(QM_ERR_DIMENSION_OVERFLOW, "rows * stride");
    if (!aligned(t.in, 2) || !aligned(t.out, 2)) return fail(QM_ERR_MISALIGNED, "q and q_out need 2-byte alignment");
    qvec = a.rotary_dim % (interleaved ? 8 : 16) == 0 && D % 8 == 0 && rows->offset % 8 == 0 && aligned(t.in, 16) &&
           aligned(t.out, 16) && (total == 1 || (t.in_stride % 8 == 0 && t.out_stride % 8 == 0));
    const Extent out = extent(t.out, t.out_stride, qwidth, total);
    if (overlap(out, extent(a.k, a.k_stride, width, total)) || overlap(out, extent(a.v, a.v_stride, width, total)) ||
        (!(t.in == t.out && t.in_stride == t.out_stride) && overlap(out, extent(t.in, t.in_stride, qwidth, total))) ||
        (a.positions && overlap(out, extent(a.positions, 2 * total, 2 * total, 1))))
      return fail(QM_ERR_INVALID_ARGUMENT, "q_out overlaps an input");
    units += total + kQueryGroups;
  }
  if (units > kv_append_most(s0->dp)) return fail(QM_ERR_DIMENSION_OVERFLOW, "rows * heads pass one launch");
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(rt, "append");
  if (st != QM_OK) return st;
  // Growth first: once a launch's sequences are committed nothing but the launch
  // itself can fail.
  for (uint32_t b = 0; b < B; ++b)
    if ((st = kv_grow(seqs[b], (uint64_t)seqs[b]->length + counts[b])) != QM_OK) return st;
  for (uint32_t b = 0; b < B; ++b)
    if ((st = stream_after(rt, seqs[b]->rt)) != QM_OK) return st;
  a.kv_heads = KVH;
  a.head_dim = D;
  a.head_dim_pad = s0->dp;
  uint32_t row0 = 0;
  for (uint32_t b0 = 0; b0 < B; b0 += kMaxAppendSeqs) {
    a.n_seqs = std::min(kMaxAppendSeqs, B - b0);
    for (uint32_t i = 0; i < a.n_seqs; ++i) {
      qm_kv* kv = seqs[b0 + i];
      KvAppendSeq& s = a.seqs[i];
      s = KvAppendSeq{};
      s.p = pages_of(kv);
      s.start = kv->length;
      s.rows = counts[b0 + i];
      s.row0 = row0;
      row0 += s.rows;
      plan_pages(kv, s.start, s.start + s.rows, &s.new_page_first, &s.new_page_count, &s.new_page_id);
      commit_pages(kv, s.new_page_first, s.new_page_count);
      kv->length += s.rows;
    }
    const hipError_t e = launch_kv_append(a, s0->bits, interleaved, vec, qvec, rt->stream);
    if (e != hipSuccess) {
      for (uint32_t i = 0; i < a.n_seqs; ++i) {
        qm_kv* kv = seqs[b0 + i];
        kv->length = a.seqs[i].start;
        rollback_pages(kv, a.seqs[i].new_page_first, a.seqs[i].new_page_count);
      }
      return hip_check(e, "append launch");
    }
  }
  for (uint32_t b = 0; b < B; ++b)
    if ((st = stream_after(seqs[b]->rt, rt)) != QM_OK) return st;
  return QM_OK;
}

qm_status qm_kv_load(qm_runtime* rt, const qm_kv* kv, uint32_t first, uint32_t count, uint16_t* k, uint16_t* v) {
  if (!rt || !kv || (!k && !v)) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (count == 0) return fail(QM_ERR_EMPTY_DIMENSION, "count must be > 0");
  if ((uint64_t)first + count > kv->length)
    return fail(QM_ERR_INVALID_SEQUENCE_LENGTH, "tokens %u .. of a sequence of %u", first, kv->length);
  if (!aligned(k, 2) || !aligned(v, 2)) return fail(QM_ERR_MISALIGNED, "k and v need 2-byte alignment");
  if (kv->rt->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "the cache is on another device");
  if (((uint64_t)count / 16 + 2) * kv->kv_heads > kv_load_most(kv->dp))
    return fail(QM_ERR_DIMENSION_OVERFLOW, "tokens * kv_heads pass one launch");
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(rt, "reading cached rows");
  if (st != QM_OK) return st;
  if ((st = stream_after(rt, kv->rt)) != QM_OK) return st;
  KvLoadArgs a{};
  a.p = pages_of(kv);
  a.k = k;
  a.v = v;
  a.first = first;
  a.count = count;
  a.kv_heads = kv->kv_heads;
  a.head_dim = kv->head_dim;
  a.head_dim_pad = kv->dp;
  const hipError_t e = launch_kv_load(a, kv->bits, rt->stream);
  if (e != hipSuccess) return hip_check(e, "cache read launch");
  return stream_after(kv->rt, rt);
}

}  // extern "C"
