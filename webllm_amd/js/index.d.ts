// Types of the Node host for libqlinear (index.js), for the reference's TypeScript code.

export interface QwenConfig {
    vocabSize: number; blockSize: number; nLayer: number; nHead: number; nKvHead: number;
    nEmbd: number; intermediate: number; rmsEps?: number; ropeTheta?: number;
}
export const QWEN25_05B: Readonly<QwenConfig>;
export function qwenHeadDim(c: QwenConfig): number;
export function qwenKvDim(c: QwenConfig): number;

export type SafetensorDtype = 'F64' | 'F32' | 'F16' | 'BF16' | 'I64' | 'I32' | 'I16' | 'I8' | 'U8' | 'BOOL';
export interface SafetensorEntry { dtype: SafetensorDtype; shape: number[]; data_offsets: [number, number]; }
export interface SafetensorFile { buffer: Uint8Array; dataStart: number; header: Record<string, SafetensorEntry>; }
export function dtypeByteSize(dtype: SafetensorDtype): number;
export function parseSafetensorsHeader(headerBytes: Uint8Array): Record<string, SafetensorEntry>;
export function parseSafetensors(buffer: ArrayBuffer | Uint8Array): SafetensorFile;
export function tensorCount(entry: SafetensorEntry): number;
export function requireTensor(file: SafetensorFile, name: string): SafetensorEntry;
export function expectTensor(file: SafetensorFile, name: string, dtype: SafetensorDtype, shape: readonly number[]): SafetensorEntry;
export function f16BitsToF32(bits: number): number;
export function readTensorBytes(file: SafetensorFile, name: string): Uint8Array;
export function readTensorF32(file: SafetensorFile, name: string): Float32Array;

/** Error thrown by the library: `code` is 'QL_E_*'. */
export interface QlError extends Error { code: string; }

export interface GptqDesc {
    qweightOff: number; qzerosOff: number | null; scalesOff: number; biasOff: number | null;
    K: number; N: number; group: number; bits: number;
}
export function makeDesc(qweightOff: number, qzerosOff: number | null, scalesOff: number, K: number,
                         N: number, group?: number, biasOff?: number | null, bits?: number): GptqDesc;

export class ArenaLayout { used: number; take(nbytes: number, align?: number): number; }
export class Arena {
    readonly size: number;
    write(off: number, data: ArrayBufferView): void;
    read<T extends ArrayBufferView>(off: number, into: T): T;
    release(): void;
}
export interface SeqInfo {
    linears: number; passes: number; tiles: number; reduces: number; grid: number;
    maxSplit: number; ldsBytes: number; deviceBytes: number;
    /** block-groups (64 columns x one group) in total and on the busiest workgroup */
    totalUnits: number; busiestUnits: number;
    /** 0: dependency-ordered tiles, 1: column strips; split: waves per 64-column block of a strip */
    kernel: number; split: number;
}
/** A forward's decode linears (M <= 16) as one persistent launch; linear i reads linear j's
 *  output when xOffs[i] === yOffs[j]. */
export class Seq {
    readonly info: SeqInfo;
    run(): void;
    status(): void;
    destroy(): void;
}
/** Elementwise work folded into one linear of a fused sequence (ql_seq_fuse). */
export interface SeqFuse {
    normWOff?: number | null; normEps?: number; x2Off?: number | null; resOff?: number | null;
}
export class Context {
    constructor(device?: number);
    seq(descs: GptqDesc[], weights: Arena, act: Arena, xOffs: number[], xDtype: number, M: number,
        yOffs: number[], fuse?: (SeqFuse | null)[]): Seq;
    info(): { name: string; cuCount: number; hbmBytes: number };
    arena(bytes: number): Arena;
    sync(): void;
    timerStart(): void;
    timerStop(): number;
    destroy(): void;
}

export interface GptqInt4Params {
    qweight: Uint8Array; qzeros?: Uint8Array | null; scales: Float32Array;
    inFeatures: number; outFeatures: number; groupSize?: number; bits?: number;
}
/** quant.ts dequantizeGptqInt4, computed on the GPU: fp32 [outFeatures, inFeatures], for any f32 scales. */
export function dequantizeGptqInt4(params: GptqInt4Params, ctx?: Context): Float32Array;

export type TensorDtype = 'f32' | 'f16' | 'u32' | 'i32' | 'u64';
export class Tensor {
    readonly arena: Arena; readonly offset: number; readonly length: number;
    readonly shape: number[]; readonly dtype: TensorDtype;
    read(): Float32Array | Uint16Array | Uint32Array | Int32Array | BigUint64Array;
    write(data: ArrayBufferView): void;
}
export class ActivationArena {
    constructor(ctx: Context, bytes: number);
    alloc(shape: number[], dtype?: TensorDtype): Tensor;
    scratchOffset(nbytes: number): number;
    reset(): void;
    release(): void;
}
export interface GptqLinearUpload {
    qweight: Uint8Array; qzeros?: Uint8Array | null; scalesF16: Uint8Array | Uint16Array;
    inFeatures: number; outFeatures: number; groupSize?: number; bias?: Float32Array | null;
}
export class QuantLinearModel {
    constructor(ctx: Context, weightCapacity: number);
    readonly weightBytes: number;
    uploadGptqLinear(name: string, p: GptqLinearUpload): void;
    uploadF32(name: string, data: ArrayLike<number>): void;
    uploadF16Bits(name: string, bytes: ArrayBufferView, shape: number[]): void;
    /** QwenGpt.gemm: C[M,N] = A[M,K] @ W^T (+ bias). */
    gemm(A: Tensor, weight: string, C: Tensor, bias: string | null, M: number, N: number, K: number): void;
    gemmBatch(A: Tensor, weights: string[], Cs: Tensor[], M: number): void;
    /** out[M, C] = the fp16 table's rows tokens[0..M) as f32 (ql_embed_f16); ids >= vocab give zeros. */
    embed(tokens: Tensor, out: Tensor, M: number, weight?: string): void;
    /** y = rmsnorm(x (+ residual)) * weight, the sum stored in sumOut (one launch: ql_add_rmsnorm). */
    rmsnorm(x: Tensor, weight: string, y: Tensor, M: number, C: number, eps: number,
            residual?: Tensor | null, sumOut?: Tensor | null): void;
    /** out = silu(gate) * up (ql_silu_mul). */
    siluMul(gate: Tensor, up: Tensor, out: Tensor, n: number): void;
    /** cosines and sines of positions 0 .. maxPos - 1 in the weight arena (ql_rope_table), named 'rope' by default */
    makeRopeTable(maxPos: number, rotDim: number, theta: number, name?: string): void;
    /** log probabilities of given tokens, entropies and top alternatives of M rows of V logits (ql_token_logprobs); T and k are the
     * tensors' second dimension */
    tokenLogprobs(logits: Tensor, M: number, V: number, o: {
        tokens?: Tensor | null; logprobs?: Tensor | null; entropy?: Tensor | null; topIds?: Tensor | null; topLogprobs?: Tensor | null;
    }): void;
    /** low-rank adapters of a linear: a fp16 bits [n, rank, K], b fp16 bits [n, N, rank], scale [n] (left out: 1) */
    uploadLora(weight: string, a: Uint16Array, b: Uint16Array, n: number, rank: number, scale?: ArrayLike<number> | null): void;
    /** each C += scale * (A . a^T) . b^T by each row's id (i32 [M]; -1: none), up to 8 linears (ql_lora_add) */
    loraAdd(A: Tensor, weights: string[], ids: Tensor, Cs: Tensor[], M: number): void;
    unpackF16(name: string, out: Tensor): void;
    /** fp16 [N,K] copies of many weights in a few launches (ql_unpack_f16_batch). */
    unpackAllF16(names: string[], outs: Tensor[]): void;
    dequantize(name: string): Float32Array;
    release(): void;
}

/** masks (ceil(M/64) words a row) and depths of a drafted tree; parents[m] is -1 or an earlier row (ql_tree_masks) */
export function treeMasks(parents: ArrayLike<number>): { masks: BigUint64Array; depths: Int32Array };

/** Per-layer K/V caches and attention (qwen.ts:200-205, :427-440); 'f16' caches take rotateStore and attendTree only. */
export class KvCache {
    constructor(ctx: Context, config: QwenConfig, dtype?: 'f32' | 'f16');
    readonly D: number;
    readonly rowLen: number;
    store(layer: number, k: Tensor, v: Tensor, rows: number, pos0: number): void;
    attend(layer: number, q: Tensor, out: Tensor, M: number, pastLen: number): void;
    /** norms (where named), rotation by positions (i32; outside the table: padding, left out) and cache store in one launch (ql_qk_norm_rope) */
    rotateStore(layer: number, model: QuantLinearModel, q: Tensor, k: Tensor, v: Tensor, positions: Tensor, qOut: Tensor, M: number,
                slot0: number, options?: { rope?: string; qNorm?: string; kNorm?: string; eps?: number }): void;
    /** attention of M <= 256 drafted rows (ql_attention_tree); masks: treeMasks' words, or none for causal rows */
    attendTree(layer: number, q: Tensor, out: Tensor, M: number, pastLen: number, masks?: Tensor | null): void;
    /** keeps an accepted path (i32 rows of the tree at pastLen) in every layer (ql_kv_move) */
    accept(pastLen: number, path: Tensor, n: number): void;
    /** the first rows of every layer into another cache (ql_kv_move); one of another context: waits for its stream and for the copy */
    fork(to: KvCache, rows: number): void;
    release(): void;
}

/** QL_DTYPE_F8: e4m3 values under powers of two (paged caches) */
export const QL_DTYPE_F8: 2;
/** A pass's rows of several sequences (PagedKvCache.batch): M rows of the tensors, `rows` of them the sequences'. */
export interface Batch {
    desc: { rowStartOff: number; kvLenOff: number; pagesOff: number; nSeq: number; maxPages: number; maxRows: number; maxLen: number };
    M: number; rows: number; tables: Tensor[];
}
/** K and V of many sequences in pages of 64, 128 or 256 tokens, fp16 or e4m3 under powers of two; sequences are numbers. */
export class PagedKvCache {
    constructor(ctx: Context, config: QwenConfig, pages: number, pageSize?: 64 | 128 | 256, dtype?: 'f16' | 'f8');
    readonly D: number;
    readonly rowLen: number;
    readonly freePages: number;
    newSequence(): number;
    length(sequence: number): number;
    free(sequence: number): void;
    cut(sequence: number, tokens: number): void;
    /** a sequence that continues another one: whole pages shared, the last one copied (ql_kv_move) */
    fork(sequence: number): number;
    /** takes the pages of a pass's rows and counts its tokens: once a pass, before its layers */
    batch(pool: ActivationArena, sequences: [number, number][], M?: number): Batch;
    /** norms (where named), rotation by the rows' positions, k and v to their pages (ql_paged_append) */
    append(layer: number, model: QuantLinearModel, q: Tensor, k: Tensor, v: Tensor, batch: Batch, qOut: Tensor,
           options?: { rope?: string; qNorm?: string; kNorm?: string; eps?: number }): void;
    /** causal GQA attention of the batch's rows over their sequences (ql_paged_attention); q and out both f32 or both f16 */
    attend(layer: number, q: Tensor, out: Tensor, batch: Batch): void;
    release(): void;
}

/** qwen-loader.ts:29-38, plus this host's config / groupSize and path / buffer alternatives to url. */
export interface QwenLoadOptions {
    /** a local path or file:// URL; default QWEN_LOCAL_DIR + 'model.safetensors' */
    url?: string;
    onProgress?: (done: number, total: number, label: string) => void;
    keepLayer?: number;
    keepEmbedRows?: { start: number; rows: number };
    path?: string; buffer?: ArrayBuffer | Uint8Array; config?: QwenConfig; groupSize?: number;
}
/** qwen-loader.ts:40-52, plus storedZeros: {nibble: count} of the stored qzeros (qwen-format.ts:112-123). */
export interface QwenLoadResult {
    gpuBytes: number; tensorCount: number; fileBytes: number;
    layer?: Record<'qW' | 'kW' | 'vW' | 'oW' | 'gateW' | 'upW' | 'downW', Float32Array>;
    embedRows?: Float32Array;
    storedZeros: Record<number, number>;
}
export const QWEN_LOCAL_DIR: string;
export function qwenLinearShapes(c: QwenConfig): Record<string, [number, number]>;
/** Rejects (throws asynchronously) on a malformed file, wrong shapes or a non-identity g_idx. */
export function loadQwenWeights(ctx: Context | null, model: QuantLinearModel, options?: QwenLoadOptions): Promise<QwenLoadResult>;
export function urlToPath(url: string): string;
export function readF16Rows(file: SafetensorFile, name: string, rowStart: number, rowCount: number, rowLength: number): Float32Array;
export function checkGIdx(file: SafetensorFile, prefix: string, inFeatures: number, group: number): void;
export function countStoredZeros(qzeros: Uint8Array, groups: number, outFeatures: number, counts: number[]): number[];
