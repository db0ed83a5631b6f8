// Internal declarations shared by the kernels and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hotarubi_gpu.h"

namespace hb {

constexpr uint32_t kAbufWord = 132;  // ISS ABUF word (memories.hpp:20)
constexpr uint32_t kWbufWord = 144;  // ISS WBUF word (memories.hpp:21)
constexpr uint32_t kDdrWord = 144;   // ABUF/WBUF word in DDR
constexpr uint32_t kAbufDepth = 8192, kWbufDepth = 2048, kFbufDepth = 4096;
constexpr uint32_t kPbufDepth = 512, kTbufDepth = 1024;
constexpr uint32_t kAddrMask = (1u << 20) - 1u;
constexpr uint32_t kMaxOps = HB_MAX_EP_OPS;
constexpr uint32_t kMaxPieces = HB_MAX_PIECES;

// Everything a GEMM tile kernel needs, passed by value.
struct GemmArgs {
  // operands: ISS images (instruction level) or DDR words (linear level)
  const uint8_t* a;
  const uint8_t* w[2];
  uint32_t* c;          // FBUF image, or fp32 bits row-major [m][n]
  uint32_t quads;       // quads of A (tile rows = 4 * quads)
  uint32_t groups;      // 8-column groups
  uint32_t m;           // linear: rows stored; instruction: 4 * quads
  uint32_t n;           // linear: columns; instruction: 8 * groups
  // instruction addressing (gemm_array.cpp:123-147)
  uint32_t a_base, a_stride, w_base, w_stride, c_base;
  // linear addressing: W word (grp, blk) at grp * kb_total + blk, A word
  // (q, blk) at q * a_row + blk
  uint32_t kb_total;
  uint32_t a_row;
  // fold schedule: pieces outer, planes inner, blocks innermost
  uint32_t n_pieces;
  uint32_t piece_off[kMaxPieces];
  uint32_t piece_kb[kMaxPieces];
  uint32_t n_planes;
  uint32_t modes[2];
  uint32_t total_steps;
  uint32_t acc;  // start from C (instruction acc / linear onto)
  // epilogue (linear level)
  uint32_t n_ops;
  uint32_t op_kind[kMaxOps];
  uint32_t op_imm[kMaxOps];
  const uint32_t* op_vec[kMaxOps];
  const uint32_t* op_x2[kMaxOps];
  const uint64_t* tbuf;
  uint8_t* q_out;     // MXINT8 DDR words [quads][n/32] or null
  // batched linear: per-layer strides (bytes / elements), 0 for one layer
  uint64_t a_batch, w_batch, c_batch, q_batch;
  uint64_t op_vec_batch[kMaxOps], op_x2_batch[kMaxOps];  // elements
  // tile grid (x: column tiles, y: row tiles, z: layers or K splits), 1-D
  uint32_t gx, gy, gz;
  // Deferred epilogue (linear level, one layer): when ws is set the GEMM
  // kernels write their raw fold results, rows [0, 4*quads), row-major
  // [split][4*quads][n], and EpilogueKernel finishes (sum over splits, -0,
  // ops, C, requantize).  K splits (fast mode): split s covers the steps
  // [s * split_steps, (s + 1) * split_steps).  With splits > 1 the kernels
  // also write one flag per (split, tile), after the sums, [split][gy][gx]
  // (tiles of tile_rows x 256): set when the split's scale bytes leave the
  // fast path's window, and the epilogue then recomputes the tile's
  // outputs exactly.
  float* ws;
  uint32_t splits, split_steps, tile_rows;
  // epilogue arithmetic of a fast-mode layer: FP32 hardware operations
  // instead of the VEC lane formulas (EpApplyFast)
  uint32_t fast_ep;
  // W planes in the panel layout (HB_LINEAR_PANELS) instead of DDR words;
  // w_steps = ceil(kb_total / 2), the steps of a panel
  uint32_t w_panels, w_steps;
  // W8 layer over FP6 W8 panels (HB_LINEAR_W8_PANELS): w[0] = w[1] = the
  // panels of both planes
  uint32_t w_fp6;
  // tile order of BandTile: column tiles in bands of this width (0: LogicalTile)
  uint32_t band;
  // A holds MXFP8 E4M3 codes (HB_LINEAR_A_FP8; one MXFP4 weight plane)
  uint32_t a_fp8;
};

// Weight panels (hb_pack_weights): one plane of n columns x kb_total
// blocks as ceil(n / 64) panels of 64 columns, each ceil(kb_total / 2)
// steps of 2 blocks; chunk (panel p, step s) is kPanelChunk bytes at
// (p * steps + s) * kPanelChunk: the 16-byte column-blocks (the DDR word's
// 16 bytes of one column: element 2j in the low nibble of byte j) at
// (b * 64 + c) * 16 for block 2s + b and column 64p + c, then the scale
// bytes at 2048 + 2 (b * 32 + c % 32) + c / 32.  Columns past n and blocks
// past kb_total are zero codes with scale byte 127.
constexpr uint32_t kPanelCols = 64, kPanelChunk = 2176, kPanelScales = 2048;

// Byte offsets of W data relative to a plane's base, split into a part that
// depends on the column only (per lane) and one on the block only (uniform):
// column col's 16 code bytes of block blk are at codes + BlockCodes(blk),
// the aligned dword holding its scale byte at scale + BlockScale(blk), the
// byte at bit `shift` of that dword.
struct WLaneOff {
  uint32_t codes, scale, shift;
};
// `panels` is g.w_panels; kernels that know the layout at compile time pass
// it as a constant (the other layout's arithmetic then disappears).
__host__ __device__ __forceinline__ WLaneOff WLane(const GemmArgs& g, uint32_t col, bool panels) {
  WLaneOff o;
  if (panels) {
    const uint32_t base = (col / kPanelCols) * g.w_steps * kPanelChunk, c = col % kPanelCols;
    o.codes = base + c * 16;
    o.scale = base + kPanelScales + 4 * ((c % 32) / 2);
    o.shift = 8 * (2 * (c % 2) + c / 32);
  } else {
    const uint32_t base = (col / 8) * g.kb_total * kDdrWord, cl = col % 8;
    o.codes = base + cl * 16;
    o.scale = base + 128 + (cl & 4);
    o.shift = 8 * (cl & 3);
  }
  return o;
}
__host__ __device__ __forceinline__ WLaneOff WLane(const GemmArgs& g, uint32_t col) {
  return WLane(g, col, g.w_panels != 0);
}
__host__ __device__ __forceinline__ uint32_t WBlockCodes(const GemmArgs& g, uint32_t blk, bool panels) {
  return panels ? (blk / 2) * kPanelChunk + (blk % 2) * (kPanelCols * 16) : blk * kDdrWord;
}
__host__ __device__ __forceinline__ uint32_t WBlockCodes(const GemmArgs& g, uint32_t blk) {
  return WBlockCodes(g, blk, g.w_panels != 0);
}
__host__ __device__ __forceinline__ uint32_t WBlockScale(const GemmArgs& g, uint32_t blk, bool panels) {
  return panels ? (blk / 2) * kPanelChunk + (blk % 2) * kPanelCols : blk * kDdrWord;
}
__host__ __device__ __forceinline__ uint32_t WBlockScale(const GemmArgs& g, uint32_t blk) {
  return WBlockScale(g, blk, g.w_panels != 0);
}
// Bytes of one plane.
inline uint64_t PanelBytes(uint32_t n, uint32_t kb_total) {
  return (uint64_t)((n + kPanelCols - 1) / kPanelCols) * ((kb_total + 1) / 2) * kPanelChunk;
}

// W8 panels (hb_pack_w8): both nibble planes of a W8 layer as the matrix
// cores' B operands, FP6 E2M3 codes of v / 2 for each nibble value v (hi
// plane -8..7, lo plane 0..15), 32 codes (a column's block) in 6 dwords as
// v_cvt_scalef32_pk32_fp6_f16 packs them.  Panel p of 64 columns is
// ceil(kb_total / 2) chunks of kW8Chunk bytes, chunk (p, s) at
// (p * steps + s) * kW8Chunk holding blocks 2s + b, b = 0, 1; with
// i = (b * 2 + l) * 64 + c for plane l (0 hi, 1 lo) and column 64p + c:
//   i * 16:              dwords 0..3 of the column-block's codes;
//   kW8Part8 + i * 8:    dwords 4..5;
//   kW8Scales + (b * 32 + c % 32) * 4 + 2 (c / 32) + l: its scale byte
//                        minus 1 (hi) or 5 (lo), modulo 256.
// Columns past n and blocks past kb_total are zero codes with scale 127.
// After the chunks, one dword per panel, at W8FlagsOffset: nonzero when a
// scale byte of the panel is outside [70, 179] (the fast path's window).
constexpr uint32_t kW8Chunk = 6400, kW8Part8 = 4096, kW8Scales = 6144;
inline uint64_t W8FlagsOffset(uint32_t n, uint32_t kb_total) {
  return (uint64_t)((n + kPanelCols - 1) / kPanelCols) * ((kb_total + 1) / 2) * kW8Chunk;
}
inline uint64_t W8PanelBytes(uint32_t n, uint32_t kb_total) {
  const uint64_t flags = (uint64_t)((n + kPanelCols - 1) / kPanelCols) * 4;
  return W8FlagsOffset(n, kb_total) + (flags + 15) / 16 * 16;
}

// Byte size of the deferred-epilogue workspace of `args` (sums and flags).
// Every workspace (the context's, and the no-allocation scratch) starts with
// kSplitCounters tile counters of the single-launch split kernel, zero
// whenever no launch is in flight (each launch puts back what it used);
// the rest, from kSplitCounterBytes on, holds a launch's partial sums.
constexpr uint32_t kSplitCounters = 4096;
constexpr size_t kSplitCounterBytes = kSplitCounters * sizeof(uint32_t);
// Partial-sum tiles a single-launch split layer may use (each 32 x 32 FP32
// plus a flag): keeps its workspace within 8 MiB.
constexpr uint32_t kSplitMaxPartials = 2040;
inline size_t WorkspaceBytes(const GemmArgs& args) {
  const size_t sums = (size_t)args.splits * args.quads * 4 * args.n * sizeof(float);
  return sums + (args.splits > 1 ? (size_t)args.splits * args.gx * args.gy * sizeof(uint32_t) : 0);
}
__device__ __forceinline__ uint32_t* SplitFlags(const GemmArgs& g) {
  return reinterpret_cast<uint32_t*>(g.ws + (size_t)g.splits * g.quads * 4 * g.n);
}

// Device scratch owned by a context, grown on demand.  A buffer, once
// handed to a kernel, is never freed before the context is destroyed: work
// still queued, and HIP graphs captured earlier, keep the address they were
// given.  Growing allocates a larger buffer and retires the old one.
struct Workspace {
  float* ptr = nullptr;
  size_t bytes = 0;
  float* retired[64] = {};  // superseded buffers, freed with the context
  uint32_t n_retired = 0;
};
// Make ws at least `bytes` long (hipMalloc; no stream synchronization).
hipError_t GrowWorkspace(Workspace& ws, size_t bytes, hipStream_t stream);
// Free the current and every retired buffer.
void FreeWorkspace(Workspace& ws);

// Workgroup -> tile mapping.  The hardware deals workgroups round-robin over
// the 8 XCDs, each with its own L2; remapping puts consecutive logical tiles
// (x fastest, then y, then layer z) on one XCD, so the workgroups that share
// a layer's weights and activations share an L2 (XcdLogical).
constexpr uint32_t kXcds = 8;
struct TileId {
  uint32_t x, y, z;
};
// Any count of workgroups: XCD x (blocks b with b % 8 == x, the hardware's
// deal) takes the contiguous run of logical indices [x q + min(x, r),
// + q + (x < r)), q = total / 8, r = total % 8 -- a bijection, so the
// logical neighbours of a block sit on its XCD and share its L2.
__device__ __forceinline__ uint32_t XcdLogical(uint32_t b, uint32_t total) {
  const uint32_t x = b % kXcds, q = total / kXcds, r = total % kXcds;
  return x * q + min(x, r) + b / kXcds;
}

__device__ __forceinline__ TileId LogicalTile(uint32_t gx, uint32_t gy, uint32_t gz) {
  const uint32_t l = XcdLogical(blockIdx.x, gx * gy * gz);
  TileId t;
  t.x = l % gx;
  t.y = (l / gx) % gy;
  t.z = l / (gx * gy);
  return t;
}

// Tile order for grids that re-read operands: logical tiles run over bands
// of `band` column tiles, row tiles within a band, so the contiguous run of
// tiles an XCD takes (XcdLogical) is about run / band row tiles by `band`
// column tiles -- a rectangle, whose A rows and W columns its L2 fetches once.
__device__ __forceinline__ TileId BandTile(uint32_t gx, uint32_t gy, uint32_t gz, uint32_t band) {
  const uint32_t l = XcdLogical(blockIdx.x, gx * gy * gz);
  band = band ? band : gx;  // 0: whole rows of column tiles, as LogicalTile
  const uint32_t per = gx * gy, li = l % per, b0 = li / (gy * band) * band;
  const uint32_t w = min(band, gx - b0), in = li - b0 * gy;
  TileId t;
  t.x = b0 + in % w;
  t.y = in / w;
  t.z = l / per;
  return t;
}
// The band width that minimizes the A and W bytes the XCDs fetch: an XCD's
// run of about tiles / 8 is rows x band, fetching rows x a_tile + band x
// w_tile (a_tile, w_tile: the A bytes of a row tile, the W bytes of a column
// tile).
uint32_t BandFor(uint32_t gx, uint32_t gy, uint64_t a_tile, uint64_t w_tile);

// Launchers (hb_gemm.hip).
hipError_t LaunchGemmInstr(const GemmArgs& args, hipStream_t stream);
hipError_t LaunchGemmInstrAliased(const GemmArgs& args, hipStream_t stream);
// Linear layer: picks the kernel, and for a single small fast layer (few
// tiles) K splits and the deferred element-parallel epilogue, in which case
// it may grow `ws` (GrowWorkspace).
// A fixed scratch buffer in place of the context's growable workspace:
// the launch never allocates; *need reports the bytes a layer needs.
struct FixedScratch {
  void* ptr;
  size_t bytes;
  size_t need;
};
hipError_t LaunchLinear(const GemmArgs& args, uint32_t batch, bool fast, Workspace& ws,
                        hipStream_t stream, FixedScratch* fixed = nullptr);
// Fast path (hb_fast.hip): block-scaled f8f6f4 MFMA for one FP4 plane or
// the W8 planes (hi, lo), in that order.
bool FastEligible(const GemmArgs& args);
// Tile grid of the fast kernel for `args` in a launch of `layers` such
// layers: column tiles, row tiles, rows per tile.
void FastGrid(const GemmArgs& args, uint32_t layers, uint32_t* gx, uint32_t* gy,
              uint32_t* tile_rows);
// Launches the fast kernel over args.gx x args.gy tiles of args.tile_rows
// rows (FastGrid's) and `batch` layers or K splits.
hipError_t LaunchLinearFast(const GemmArgs& args, uint32_t batch, hipStream_t stream);
// Streaming MXFP4 kernel (hb_fast4.hip) for 128-row tiles of plain layers
// (no ops, no requantize, no K splits); `args` carries the tile grid.
bool Fp4Eligible(const GemmArgs& args, uint32_t tile_rows);
hipError_t LaunchFp4(const GemmArgs& args, hipStream_t stream);
// MXFP4 layers of independent waves (hb_wave.hip): one piece, every
// epilogue.  WaveColumns: the columns of a wave's tile (128 or 64), or 0 where
// another kernel takes the launch.
uint32_t WaveColumns(const GemmArgs& args, uint32_t batch);
hipError_t LaunchWave(const GemmArgs& args, uint32_t batch, uint32_t columns, hipStream_t stream);
// Streaming kernel over weight panels (hb_panel.hip): fast MXFP4, plain
// layers of more than 64 rows, one piece over every block.
bool PanelEligible(const GemmArgs& args);
hipError_t LaunchPanel(const GemmArgs& args, uint32_t batch, hipStream_t stream);
// Streaming kernel over weight panels with a global-to-LDS ring (hb_stream.hip).
bool StreamEligible(const GemmArgs& args);
hipError_t LaunchStream(const GemmArgs& args, uint32_t batch, hipStream_t stream);
// W8 layers over FP6 W8 panels (hb_w8.hip): every shape, both modes (exact
// mode folds each output exactly).
hipError_t LaunchW8Linear(const GemmArgs& args, uint32_t batch, bool fast, hipStream_t stream);
// The W8 DDR planes (hi, lo) <-> W8 panels (hb_w8.hip).
hipError_t LaunchPackW8(const uint8_t* hi, const uint8_t* lo, uint32_t n, uint32_t kb_total,
                        uint8_t* out, hipStream_t stream);
hipError_t LaunchUnpackW8(const uint8_t* in, uint32_t n, uint32_t kb_total, uint8_t* hi,
                          uint8_t* lo, hipStream_t stream);
// Weight preparation (hb_prep.hip): fp32 weights -> the W8 planes' WBUF
// words; MXFP4 codes and scale bytes -> canonical WBUF words.  *bad_flag is
// set where the reference would reject the input.
hipError_t LaunchW8FromFp32(const float* w, uint32_t rows, uint32_t cols, uint32_t out_rows,
                            uint8_t* hi, uint8_t* lo, uint32_t* bad_flag, hipStream_t stream);
hipError_t LaunchMxfp4Canonical(const uint8_t* codes, const uint8_t* scales, uint32_t rows,
                                uint32_t cols, int32_t exponent_shift, uint32_t out_rows,
                                uint8_t* out, uint32_t* bad_flag, hipStream_t stream);
// DDR words <-> panels of one plane (hb_panel.hip).
hipError_t LaunchPackPanels(const uint8_t* w, uint32_t n, uint32_t kb_total, uint8_t* out,
                            hipStream_t stream);
hipError_t LaunchUnpackPanels(const uint8_t* in, uint32_t n, uint32_t kb_total, uint8_t* w,
                              hipStream_t stream);
// Fast path for layers of at most 64 rows (hb_skinny.hip): split-K over the
// waves of a workgroup, W streamed into registers.
hipError_t LaunchLinearSkinny(const GemmArgs& args, uint32_t batch, hipStream_t stream);
// One fast layer of at most kSplitMaxRows rows in one launch: 32 x 32 tiles,
// K split over workgroups, the last split of a tile finishing it.
constexpr uint32_t kSplitMaxRows = 160;
bool SplitEligible(const GemmArgs& args, uint32_t batch);
// Grid and K split of a split launch (sets gx, gy, splits, split_steps:
// splits of at least 2 steps, at most max_splits, one wave each) and the
// workspace bytes it needs past the counters (0: no partials).
constexpr uint32_t kMaxSplitWaves = 8;
// Waves a split workgroup has at least: the epilogue's 4 row groups of a
// 32 x 32 tile go to 4 finishers, one each, also where K has fewer splits
// (the waves past the splits fold nothing).
constexpr uint32_t kSplitFinishWaves = 4;
size_t SplitPlan(GemmArgs& args, uint32_t max_splits = kMaxSplitWaves);
hipError_t LaunchSplitLinear(const GemmArgs& args, hipStream_t stream);
// The same tiles for `batch` layers (int8 activations; args from SplitPlan).
hipError_t LaunchSplitBatch(const GemmArgs& args, uint32_t batch, hipStream_t stream);
// Up to kMaxGroup single-launch split layers (args from SplitPlan, one
// format) in one launch: units of one layer or a fused pair (the second's op
// x2_op reads the first's C); second[u] == kMaxGroup for a single layer;
// tile_end[u] the cumulative workgroup count.  A pair's layers fold side by
// side (their splits add up to at most kMaxSplitWaves); `waves` = the
// largest wave count of a unit.
constexpr uint32_t kMaxGroup = HB_MAX_GROUP;
// Compute units of the current device (cached per device).
int DeviceCus();
// Waves of the split kernels one CU holds at once (2 per SIMD: they take
// more than 128 VGPRs).
constexpr uint32_t kSplitWavesPerCu = 8;
struct SplitGroup {
  GemmArgs g[kMaxGroup];
  uint32_t units;
  uint32_t tile_end[kMaxGroup], first[kMaxGroup], second[kMaxGroup], x2_op[kMaxGroup];
};
hipError_t LaunchSplitGroup(const SplitGroup& grp, uint32_t waves, hipStream_t stream);
// Deferred epilogue (hb_vec.hip): reads args.ws, writes C and q_out.
hipError_t LaunchEpilogue(const GemmArgs& args, hipStream_t stream);

// DMA-engine W8 operand builders (hb_dma.hip).
hipError_t LaunchSplit8(const uint8_t* src, uint64_t stride, uint32_t rows, uint32_t row_words,
                        uint8_t* hi, uint8_t* lo, hipStream_t stream);
hipError_t LaunchRowLoad(const uint8_t* src, uint64_t stride, uint32_t rows, uint32_t row_words,
                        uint32_t tok, uint32_t token_bytes, const uint32_t* index, uint8_t* out,
                        hipStream_t stream);
hipError_t LaunchRowStore(const uint8_t* words, uint32_t rows, uint32_t row_words, uint32_t tok,
                         uint32_t token_bytes, uint8_t* dst, uint64_t stride, hipStream_t stream);
struct GaccArgs {
  const uint8_t* base;  // byte 0 of the 16-byte unit addresses
  const uint8_t* list;  // quad 0's list
  uint64_t list_stride;
  uint32_t quads, slots, blocks, w_stride, accumulate;
  float* out;           // [quads * 4][32 * blocks]
};
hipError_t LaunchGacc(const GaccArgs& a, hipStream_t stream);
hipError_t LaunchT32Split8(const uint8_t* src, uint64_t stride, uint32_t rows, uint32_t row_words,
                           uint8_t* hi, uint8_t* lo, hipStream_t stream);

// VEC (hb_vec.hip).
struct VecPass {
  uint32_t src, src2, d;   // register values (src, src2 masked to 12 bits)
  uint32_t x2_en;
  uint32_t c0;             // 0 zero, 1 x2, 2 pbuf
  uint32_t b;              // 0 one, 1 x2, 2 pbuf, 3 imm
  uint32_t act;            // nl = ACT
  uint32_t po;             // 0 add, 1 max, 2 signfix
  uint32_t pv;             // c1 = x2
  uint32_t to_abuf;        // final pass with quantize
  uint32_t imm;
  uint32_t pb;             // PBUF base (9 bits)
  uint32_t quads, words, n8;
};
hipError_t LaunchVecPass(const VecPass& pass, uint8_t* abuf, uint32_t* fbuf,
                         const uint32_t* pbuf, const uint64_t* tbuf, uint32_t* temp,
                         hipStream_t stream);
// fp8: MXFP8 E4M3 codes (OCP MX rule) instead of MXINT8, in the same words.
hipError_t LaunchEncodeMxint8(const float* x, uint32_t rows, uint32_t cols, uint8_t* out,
                              uint32_t* bad_flag, hipStream_t stream, bool fp8 = false);

// Row programs of the VEC library (12 SOFTMAX, 22 LAYERNORM, 34 RMSNORM):
// the register values of quad 0's slot and the per-quad steps.
struct VecRowArgs {
  uint32_t entry, quantize, rows_q, n8;
  uint32_t src, scratch, dst, dst_step;  // unmasked register values
  uint32_t pbase, quarter, aux, imm;
  uint32_t rn;  // CountReciprocal(aux)
};
constexpr uint32_t kRowSoftmax = 12, kRowLayerNorm = 22, kRowRmsNorm = 34;
// The FBUF (and PBUF) words each pass of a row program reads and writes for
// one quad, for the host's checks: up to 5 passes.
struct RowPassSpan {
  uint32_t src, dst;  // register values (masked on use)
  bool writes;        // an FBUF or final store
  bool final_;        // the program's last pass (ABUF when quantizing)
};
int RowProgramSpans(const VecRowArgs& a, uint32_t quad, RowPassSpan* out);
// The same programs over row-major DDR tensors (hb_rows): rows of the last
// quad past `rows` are zero rows whose results are not stored.
struct VecRowDdr {
  const uint32_t* x;  // fp32 [rows][cols]
  const uint32_t *gamma, *beta;  // fp32 [cols]
  uint32_t* y;        // fp32 [rows][cols] (not quantizing)
  uint8_t* q_out;     // MXINT8 DDR words [ceil(rows/4)][cols/32] (quantizing)
  uint32_t rows, cols;
};
// serial: one workgroup runs the quads in the engine's order (for programs
// whose quads share FBUF or ABUF words); otherwise one workgroup per quad.
hipError_t LaunchVecRows(const VecRowArgs& a, uint8_t* abuf, uint32_t* fbuf, const uint32_t* pbuf,
                         const uint64_t* tbuf, hipStream_t stream, bool serial);
hipError_t LaunchRowsDdr(const VecRowArgs& a, const VecRowDdr& d, const uint64_t* tbuf,
                         hipStream_t stream);

// Serving operators (hb_kv.hip, hb_attn.hip) over the paged MXFP4 cache.
struct PlanArgs {
  const int32_t *lens, *new_tokens, *free_pages, *free_count;
  int32_t *table, *cu, *kv_lens, *slots, *positions, *status;
  uint32_t batch, columns, table_stride, page, size, free_size;
};
hipError_t LaunchPlan(const PlanArgs& a, hipStream_t stream);
// Strides are elements, of a token's row and of a head.
struct RopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  uint64_t q_token, q_head, k_token, k_head, q_out_token, q_out_head, k_out_token, k_out_head;
  const float *gamma_q, *gamma_k;  // null: not normalised
  const int32_t* positions;        // [axes][position_stride]
  uint64_t position_stride;
  const double* inv_freq;          // [rot / 2]
  float eps;
  uint32_t type, tokens, q_heads, k_heads, dim, rot, neighbours;
  uint32_t sections[2];            // where the second and third axis' pairs start
  uint32_t lanes, parts;           // set by the launcher
};
hipError_t LaunchRope(const RopeArgs& a, hipStream_t stream);
struct KvRowsArgs {
  const void *k, *v;               // append
  void *k_out, *v_out;             // read
  uint64_t k_token, k_head, v_token, v_head;
  const int32_t* slots;
  uint8_t* cache;
  uint32_t type, tokens, pages, heads, groups, dim;
  uint32_t vec;                    // set by the launcher
};
// tokens * heads < 2^31
hipError_t LaunchKvRows(const KvRowsArgs& a, bool read, hipStream_t stream);
struct AttnArgs {
  const void* q;
  void* out;
  uint64_t q_token, q_head, out_token, out_head;  // elements
  const uint8_t* cache;
  const int32_t *table, *cu, *kv_lens, *prefix;   // prefix may be null
  uint32_t type, tokens, batch, q_heads, heads, dim, pages, groups, columns, table_stride;
  uint32_t max_new, max_kv, window;
  float scale, cap;                               // cap 0: scores as they are
  // set by the launcher: tiles of rows of one (request, K/V head), splits of
  // a tile's records, records of a split, and the partial results
  uint32_t tiles, splits, split_records;
  float sign;  // of scale, which is positive then
  float* ws;
  // prompts: records of a request that are opened, and where
  uint32_t opened;
  uint8_t* opened_at;
};
// How a call is divided: HB_KV_WAY_*, 16-row tiles of a wave, tiles of a request
// and K/V head, splits of a tile's records (workgroups of the shares), records
// of a split, bytes of workspace.
struct AttnWay {
  uint32_t way, tiles_of_16, tiles, splits, split_records;
  uint64_t workspace;
};
AttnWay WayOfAttention(const AttnArgs& a);
hipError_t LaunchAttention(const AttnArgs& a, Workspace& ws, hipStream_t stream);
// Many rows of 16-bit types (hb_prompt.hip): 16-row tiles of a wave, rows of a
// workgroup, and the workspace of a launch.
uint32_t PromptTiles(uint32_t dim);
uint32_t PromptRows(uint32_t dim);
uint64_t PromptBytes(const AttnArgs& a);
hipError_t LaunchPrompt(const AttnArgs& a, Workspace& ws, hipStream_t stream);

}  // namespace hb
