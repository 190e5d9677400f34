'use strict';
/**
 * Node host for libqlinear: the reference's TypeScript surface for the GPTQ int4 path, with the
 * int4 work on the MI355X through the Node-API addon (webllm_amd/lib/qlinear_napi.node).
 *
 * Same names, argument meaning and error behaviour as (paths in the intplusplus/webllm checkout):
 *   parseSafetensors, parseSafetensorsHeader,    src/weights/safetensors.ts:40-222
 *   requireTensor, expectTensor, tensorCount,
 *   readTensorBytes, readTensorF32, f16BitsToF32,
 *   dtypeByteSize
 *   dequantizeGptqInt4(params)                   src/weights/quant.ts:42-118 (exact, on the GPU)
 *   QuantLinearModel.gemm(A, weight, C, bias,    src/model/qwen.ts:568-618 QwenGpt.gemm
 *     M, N, K)
 *   loadQwenWeights(ctx, model, options)         src/weights/qwen-loader.ts:102-177 (async), with
 *                                                the packed int4 tensors uploaded as they are
 *   readF16Rows                                  src/weights/qwen-loader.ts:70-93
 *   checkGIdx, countStoredZeros                  src/tests/qwen/qwen-format.ts:112-130 probes
 *   QWEN25_05B, qwenKvDim                        src/model/qwen-config.ts:1-54
 *
 * Errors are thrown as Error (the reference's `throw new Error(msg)`); library status codes carry
 * `err.code` = 'QL_E_*'. There is no CPU fallback: a missing addon throws at require time,
 * that of passes over many requests where it is needed first.
 */
const fs = require('fs');
const path = require('path');

const ADDON_PATH = path.join(__dirname, '..', 'lib', 'qlinear_napi.node');
if (!fs.existsSync(ADDON_PATH)) {
    throw new Error(`qlinear: addon not built at ${ADDON_PATH} (run __graft_entry__.build())`);
}
const addon = require(ADDON_PATH);
// passes over many requests, on the same handles: loaded by the first that needs it
let loadedBatchAddon = null;
function batchAddon() {
    if (!loadedBatchAddon) {
        const at = path.join(path.dirname(ADDON_PATH), 'qlinear_batch_napi.node');
        if (!fs.existsSync(at)) throw new Error(`qlinear: addon not built at ${at} (run __graft_entry__.build())`);
        loadedBatchAddon = require(at);
    }
    return loadedBatchAddon;
}

const QL_DTYPE_F32 = 0;
const QL_DTYPE_F16 = 1;
const QL_DTYPE_F8 = 2;
// most rows of a pass, sequences, tokens of one, rows times heads of q, k and v, sequences times kv heads (ql_batch_desc)
const BATCH = Object.freeze({ rows: 65535, seqs: 4096, tokens: 2 ** 26, heads: 2 ** 23, seqHeads: 2 ** 22 });

// ------------------------------------------------------------------ config (qwen-config.ts)

const QWEN25_05B = Object.freeze({
    vocabSize: 151936, blockSize: 128, nLayer: 24, nHead: 14, nKvHead: 2, nEmbd: 896,
    intermediate: 4864, rmsEps: 1e-6, ropeTheta: 1000000,
});

function qwenHeadDim(c) { return c.nEmbd / c.nHead; }
function qwenKvDim(c) { return c.nKvHead * qwenHeadDim(c); }

// ------------------------------------------------------------------ safetensors.ts

const DTYPE_BYTES = { F64: 8, I64: 8, F32: 4, I32: 4, F16: 2, BF16: 2, I16: 2, I8: 1, U8: 1, BOOL: 1 };

function dtypeByteSize(dtype) {
    const n = DTYPE_BYTES[dtype];
    if (n === undefined) throw new Error(`unknown safetensors dtype: ${dtype}`);
    return n;
}

function parseSafetensorsHeader(headerBytes) {
    let parsed;
    try {
        parsed = JSON.parse(Buffer.from(headerBytes.buffer, headerBytes.byteOffset,
            headerBytes.byteLength).toString('utf8'));
    } catch (err) {
        throw new Error(`safetensors: header JSON parse failed: ${err.message}`);
    }
    if (typeof parsed !== 'object' || parsed === null) {
        throw new Error('safetensors: header is not a JSON object');
    }
    const header = {};
    for (const name of Object.keys(parsed)) {
        if (name === '__metadata__') continue;
        const item = parsed[name];
        if (typeof item !== 'object' || item === null) throw new Error(`safetensors: ${name} entry invalid`);
        if (typeof item.dtype !== 'string') throw new Error(`safetensors: ${name} missing dtype`);
        if (!Array.isArray(item.shape)) throw new Error(`safetensors: ${name} missing shape`);
        if (!Array.isArray(item.data_offsets) || item.data_offsets.length !== 2) {
            throw new Error(`safetensors: ${name} data_offsets invalid`);
        }
        const start = Number(item.data_offsets[0]);
        const end = Number(item.data_offsets[1]);
        if (!Number.isFinite(start) || !Number.isFinite(end) || start < 0 || end < start) {
            throw new Error(`safetensors: ${name} data_offsets out of range`);
        }
        header[name] = { dtype: item.dtype, shape: item.shape.map(Number), data_offsets: [start, end] };
    }
    return header;
}

/** buffer: ArrayBuffer or Node Buffer / Uint8Array (the whole file). */
function parseSafetensors(buffer) {
    const bytes = buffer instanceof ArrayBuffer ? new Uint8Array(buffer)
        : new Uint8Array(buffer.buffer, buffer.byteOffset, buffer.byteLength);
    if (bytes.byteLength < 8) throw new Error('safetensors: buffer too short');
    const dv = new DataView(bytes.buffer, bytes.byteOffset, bytes.byteLength);
    const headerLen = dv.getUint32(0, true);
    if (dv.getUint32(4, true) !== 0) throw new Error('safetensors: header longer than 4 GiB is not supported');
    const dataStart = 8 + headerLen;
    if (headerLen <= 0 || dataStart > bytes.byteLength) {
        throw new Error(`safetensors: invalid header length headerLen=${headerLen} bufferSize=${bytes.byteLength}`);
    }
    const header = parseSafetensorsHeader(bytes.subarray(8, dataStart));
    for (const name of Object.keys(header)) {
        if (dataStart + header[name].data_offsets[1] > bytes.byteLength) {
            throw new Error(`safetensors: ${name} data out of bounds end=${header[name].data_offsets[1]}`);
        }
    }
    return { buffer: bytes, dataStart, header };
}

function tensorCount(entry) { return entry.shape.reduce((a, b) => a * b, 1); }

function requireTensor(file, name) {
    const entry = file.header[name];
    if (!entry) throw new Error(`safetensors: missing tensor ${name}`);
    return entry;
}

function expectTensor(file, name, dtype, shape) {
    const entry = requireTensor(file, name);
    if (entry.dtype !== dtype) throw new Error(`safetensors: ${name} dtype=${entry.dtype}, expected ${dtype}`);
    if (entry.shape.length !== shape.length || entry.shape.some((v, i) => v !== shape[i])) {
        throw new Error(`safetensors: ${name} shape=[${entry.shape}], expected [${shape}]`);
    }
    return entry;
}

function f16BitsToF32(bits) {
    const sign = (bits & 0x8000) !== 0 ? -1 : 1;
    const exp = (bits >>> 10) & 0x1f;
    const mant = bits & 0x03ff;
    if (exp === 0) return sign * mant * Math.pow(2, -24);
    if (exp === 31) return mant === 0 ? sign * Infinity : NaN;
    return sign * (1 + mant / 1024) * Math.pow(2, exp - 15);
}

/** Raw bytes of one tensor, as a copy (aligned for typed views). */
function readTensorBytes(file, name) {
    const entry = requireTensor(file, name);
    const start = file.dataStart + entry.data_offsets[0];
    const length = tensorCount(entry) * dtypeByteSize(entry.dtype);
    return Uint8Array.from(file.buffer.subarray(start, start + length));
}

function readTensorF32(file, name) {
    const entry = requireTensor(file, name);
    const count = tensorCount(entry);
    const start = file.dataStart + entry.data_offsets[0];
    const view = new DataView(file.buffer.buffer, file.buffer.byteOffset + start,
        entry.data_offsets[1] - entry.data_offsets[0]);
    const out = new Float32Array(count);
    const tmp = new DataView(new ArrayBuffer(4));
    for (let i = 0; i < count; i++) {
        switch (entry.dtype) {
            case 'F32': out[i] = view.getFloat32(i * 4, true); break;
            case 'F16': out[i] = f16BitsToF32(view.getUint16(i * 2, true)); break;
            case 'BF16':
                tmp.setUint32(0, view.getUint16(i * 2, true) << 16, true);
                out[i] = tmp.getFloat32(0, true);
                break;
            case 'U8': out[i] = view.getUint8(i); break;
            case 'I8': out[i] = view.getInt8(i); break;
            default: throw new Error(`readTensorF32: unsupported dtype ${entry.dtype} (${name})`);
        }
    }
    return out;
}

// ------------------------------------------------------------------ device objects

/** Bump allocator over one arena, 256-byte aligned slices (the library's alignment contract). */
class ArenaLayout {
    constructor() { this.used = 0; }
    take(nbytes, align) {
        const a = align || 256;
        const off = Math.ceil(this.used / a) * a;
        this.used = off + nbytes;
        return off;
    }
}

class Arena {
    constructor(ctx, bytes) {
        this.ctx = ctx;
        this.handle = addon.arenaReserve(ctx.handle, bytes);
        this.size = bytes;
        ctx._arenas.add(this);
    }
    write(off, typed) { addon.arenaWrite(this.handle, off, typed); }
    read(off, typed) { addon.arenaRead(this.handle, off, typed); return typed; }
    release() {
        if (this.handle) {
            addon.arenaRelease(this.handle);
            this.handle = null;
            this.ctx._arenas.delete(this);
        }
    }
}

/**
 * A forward's decode linears as one persistent launch (ql_seq_*; the CommandBatch of
 * src/gpu/pipeline.ts:71-116 with passBreak, qwen.ts:556-559): linear i consumes linear j's
 * output when xOffs[i] === yOffs[j], and the kernel orders the two on the device.
 * `fuse` (optional, one entry per linear, null for none) folds the layer's elementwise work in
 * (ql_seq_create_fused; qwen.ts:401-405, :445-478): {normWOff, normEps} normalizes the linear's
 * input (RMSNorm weights at normWOff in `weights`), {x2Off} multiplies silu(x) by a second input,
 * {resOff} adds a residual to the output. An offset equal to another linear's yOffs entry makes
 * that linear the producer.
 */
class Seq {
    constructor(ctx, descs, weights, act, xOffs, xDtype, M, yOffs, fuse) {
        this.ctx = ctx;
        this.handle = fuse
            ? addon.seqCreate(ctx.handle, descs, weights.handle, act.handle, xOffs, xDtype, M, yOffs, fuse)
            : addon.seqCreate(ctx.handle, descs, weights.handle, act.handle, xOffs, xDtype, M, yOffs);
        ctx._seqs.add(this);
    }
    get info() { return addon.seqInfo(this.handle); }
    run() { addon.seqRun(this.ctx.handle, this.handle); }
    /** Waits for the stream; throws QL_E_STATE if a run was aborted. */
    status() { addon.seqStatus(this.ctx.handle, this.handle); }
    destroy() {
        if (this.handle) {
            addon.seqDestroy(this.handle);
            this.handle = null;
            this.ctx._seqs.delete(this);
        }
    }
}

/** One device, one stream (ql_create). */
class Context {
    constructor(device) {
        this.handle = addon.create(device === undefined ? 0 : device);
        this._arenas = new Set();
        this._seqs = new Set();
    }
    seq(descs, weights, act, xOffs, xDtype, M, yOffs, fuse) {
        return new Seq(this, descs, weights, act, xOffs, xDtype, M, yOffs, fuse);
    }
    info() { return addon.deviceInfo(this.handle); }
    arena(bytes) { return new Arena(this, bytes); }
    sync() { addon.sync(this.handle); }
    timerStart() { addon.timerStart(this.handle); }
    timerStop() { return addon.timerStop(this.handle); }
    destroy() {
        for (const q of Array.from(this._seqs)) q.destroy();
        for (const a of Array.from(this._arenas)) a.release();
        if (this.handle) { addon.destroy(this.handle); this.handle = null; }
    }
}

function makeDesc(qweightOff, qzerosOff, scalesOff, K, N, group, biasOff, bits) {
    return {
        qweightOff, qzerosOff: qzerosOff === undefined ? null : qzerosOff, scalesOff,
        biasOff: biasOff === undefined ? null : biasOff, K, N,
        group: group === undefined ? 128 : group, bits: bits === undefined ? 4 : bits,
    };
}

const CODE_NAMES = {
    '-1': 'QL_E_BITS', '-2': 'QL_E_GROUP', '-3': 'QL_E_DIMS', '-4': 'QL_E_QWEIGHT_SHORT',
    '-5': 'QL_E_SCALES_SHORT', '-6': 'QL_E_QZEROS_SHORT', '-7': 'QL_E_GROUP_PACK',
};

function libError(code, message) {
    const e = new Error(`${code}: ${message}`);
    e.code = code;
    return e;
}

// ------------------------------------------------------------------ quant.ts

let defaultCtx = null;

/**
 * quant.ts:42-118: GptqInt4Params -> fp32 [outFeatures, inFeatures], computed on the GPU
 * (ql_unpack_f32_ex with the f32 scales as given: any Float32Array, quant.ts:22-23; bit-identical
 * to the reference's loop). `ctx` defaults to device 0.
 */
function dequantizeGptqInt4(params, ctx) {
    const groupSize = params.groupSize === undefined || params.groupSize === null ? 128 : params.groupSize;
    const bits = params.bits === undefined || params.bits === null ? 4 : params.bits;
    const inF = params.inFeatures;
    const outF = params.outFeatures;
    // quant.ts:46-79 order: bits, group, dims, qweight bytes, scales count, qzeros bytes, group % 8
    const shapeRc = addon.validate(makeDesc(0, null, 0, inF, outF, groupSize, null, bits), 2 ** 52);
    if (shapeRc === -1 || shapeRc === -2 || shapeRc === -3) throw libError(CODE_NAMES[shapeRc], addon.lastError());
    const need = addon.gptqSizes(inF, outF, groupSize);
    if (params.qweight.byteLength < need.qweightBytes) {
        throw libError('QL_E_QWEIGHT_SHORT', `GPTQ: qweight needs ${need.qweightBytes} bytes, got ${params.qweight.byteLength}`);
    }
    if (params.scales.length < need.scalesBytes / 2) {
        throw libError('QL_E_SCALES_SHORT', `GPTQ: scales need ${need.scalesBytes / 2} values, got ${params.scales.length}`);
    }
    const qz = params.qzeros || null;
    if (qz && qz.byteLength < need.qzerosBytes) {
        throw libError('QL_E_QZEROS_SHORT', `GPTQ: qzeros need ${need.qzerosBytes} bytes, got ${qz.byteLength}`);
    }
    if (shapeRc === -7) throw libError('QL_E_GROUP_PACK', `GPTQ: groupSize=${groupSize} must be a multiple of 8`);
    const s32 = Float32Array.from(params.scales.subarray(0, need.scalesBytes / 2));
    if (!ctx) { if (!defaultCtx) defaultCtx = new Context(0); ctx = defaultCtx; }
    const lay = new ArenaLayout();
    const oQw = lay.take(need.qweightBytes);
    const oQz = qz ? lay.take(need.qzerosBytes) : null;
    const oSc = lay.take(s32.byteLength);
    const w = ctx.arena(lay.used + 256);
    const out = ctx.arena(Math.max(inF * outF * 4, 16));
    try {
        w.write(oQw, params.qweight.subarray(0, need.qweightBytes));
        if (qz) w.write(oQz, qz.subarray(0, need.qzerosBytes));
        w.write(oSc, s32);
        addon.unpack(ctx.handle, makeDesc(oQw, oQz, oSc, inF, outF, groupSize, null, bits), w.handle,
            out.handle, 0, true, QL_DTYPE_F32);
        return out.read(0, new Float32Array(outF * inF));
    } finally {
        w.release();
        out.release();
    }
}

// ------------------------------------------------------------------ QwenGpt weight side (qwen.ts)

/** Slice of a device arena: {arena, offset, length, shape, dtype} (buffer.ts:12-18). */
class Tensor {
    constructor(arena, offset, length, shape, dtype, pool) {
        this.arena = arena; this.offset = offset; this.length = length; this.shape = shape;
        this.dtype = dtype; this.pool = pool || null;
    }
    read() {
        const T = { f16: Uint16Array, u32: Uint32Array, i32: Int32Array, u64: BigUint64Array }[this.dtype] || Float32Array;
        return this.arena.read(this.offset, new T(this.length));
    }
    write(data) { this.arena.write(this.offset, data); }
}

/** Per-step activation arena (arena.ts): bump allocation from the front, split-K scratch from the back. */
class ActivationArena {
    constructor(ctx, bytes) {
        this.arena = ctx.arena(bytes);
        this.layout = new ArenaLayout();
    }
    alloc(shape, dtype) {
        const dt = dtype || 'f32';
        const n = shape.reduce((a, b) => a * b, 1);
        const off = this.layout.take(n * (dt === 'f16' ? 2 : dt === 'u64' ? 8 : 4));
        if (this.layout.used > this.arena.size) throw new Error('activation arena exhausted');
        return new Tensor(this.arena, off, n, shape.slice(), dt, this);
    }
    scratchOffset(nbytes) {
        const off = Math.floor((this.arena.size - nbytes) / 256) * 256;
        if (off < this.layout.used) throw new Error(`activation arena: no room for ${nbytes} scratch bytes`);
        return off;
    }
    reset() { this.layout = new ArenaLayout(); }
    release() { this.arena.release(); }
}

class QuantLinearModel {
    /** Weight side of QwenGpt with GPTQ weights kept packed in one device arena, addressed by name. */
    constructor(ctx, weightCapacity) {
        this.ctx = ctx;
        this.weights = ctx.arena(weightCapacity);
        this.layout = new ArenaLayout();
        this.linears = new Map();
        this.f32Weights = new Map();
        this.f16Weights = new Map();
        this.loras = new Map();
    }
    get weightBytes() { return this.layout.used; }
    _place(typed) {
        const off = this.layout.take(typed.byteLength);
        if (this.layout.used > this.weights.size) {
            throw new Error(`weight arena exhausted (${this.layout.used} > ${this.weights.size})`);
        }
        this.weights.write(off, typed);
        return off;
    }
    /** qweight I32 [in/8, out], qzeros I32 [in/g, out/8] or null, scales F16 bits [in/g, out], bias F32 [out] or null. */
    uploadGptqLinear(name, p) {
        if (this.linears.has(name)) throw new Error(`weight already exists: ${name}`);
        const group = p.groupSize || 128;
        const qw = this._place(p.qweight);
        const qz = p.qzeros ? this._place(p.qzeros) : null;
        const sc = this._place(p.scalesF16);
        const b = p.bias ? this._place(Float32Array.from(p.bias)) : null;
        const desc = makeDesc(qw, qz, sc, p.inFeatures, p.outFeatures, group, b);
        const rc = addon.validate(desc, this.weights.size);
        if (rc !== 0) throw libError(CODE_NAMES[rc] || 'QL_E_INVALID', addon.lastError());
        this.linears.set(name, { desc, K: p.inFeatures, N: p.outFeatures });
    }
    uploadF32(name, data) {
        if (this.f32Weights.has(name)) throw new Error(`weight already exists: ${name}`);
        const a = Float32Array.from(data);
        this.f32Weights.set(name, new Tensor(this.weights, this._place(a), a.length, [a.length], 'f32'));
    }
    uploadF16Bits(name, bytes, shape) {
        if (this.f16Weights.has(name)) throw new Error(`weight already exists: ${name}`);
        const n = shape.reduce((x, y) => x * y, 1);
        this.f16Weights.set(name, new Tensor(this.weights, this._place(bytes), n, shape.slice(), 'f16'));
    }
    linear(name) {
        const l = this.linears.get(name);
        if (!l) throw new Error(`missing int4 weight: ${name}`);
        return l;
    }
    /** C[M,N] = A[M,K] @ W^T (+ bias) — qwen.ts:568-618. A f32 or f16, C f32. */
    gemm(A, weight, C, bias, M, N, K) {
        if (this.f16Weights.has(weight) && !this.linears.has(weight)) return this._gemmF16(A, weight, C, bias, M, N, K);
        const lin = this.linear(weight);
        if (lin.K !== K || lin.N !== N) throw new Error(`gemm: ${weight} is [${lin.N},${lin.K}], called with N=${N} K=${K}`);
        if (bias !== null && bias !== undefined && lin.desc.biasOff === null) throw new Error(`missing f32 weight: ${bias}`);
        let desc = lin.desc;
        if ((bias === null || bias === undefined) && desc.biasOff !== null) desc = Object.assign({}, desc, { biasOff: null });
        if (A.arena !== C.arena || !A.pool || A.pool !== C.pool) throw new Error('gemm: A and C must come from one ActivationArena');
        if (A.length < M * K || C.length < M * N) throw new Error('gemm: tensor too small for [M,K] / [M,N]');
        const plan = addon.planLinear(M, N, K, desc.group);
        const scratch = A.pool.scratchOffset(plan.scratchBytes);
        addon.linear(this.ctx.handle, desc, this.weights.handle, A.arena.handle, A.offset,
            A.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32, M, C.offset, scratch);
    }
    /** fp16 weights (the tied lm_head `embed`, qwen.ts:488-489): f32 A and C, fp32 accumulation. */
    _gemmF16(A, weight, C, bias, M, N, K) {
        const w = this.f16Weights.get(weight);
        if (w.shape[0] !== N || w.shape[1] !== K) throw new Error(`gemm: ${weight} is [${w.shape}], called with N=${N} K=${K}`);
        let b = null;
        if (bias !== null && bias !== undefined) {
            const t = this.f32Weights.get(bias);
            if (!t) throw new Error(`missing f32 weight: ${bias}`);
            b = t.offset;
        }
        if (A.dtype !== 'f32' || C.dtype !== 'f32') throw new Error('gemm over fp16 weights takes f32 A and C');
        if (A.arena !== C.arena) throw new Error('gemm: A and C must live in the same activation arena');
        if (A.length < M * K || C.length < M * N) throw new Error('gemm: tensor too small for [M,K] / [M,N]');
        addon.gemvF16w(this.ctx.handle, this.weights.handle, w.offset, b, A.arena.handle, A.offset, M, N, K, C.offset);
    }
    /** out[M, C] = rows tokens[0..M) of the fp16 table as f32 (embedding_f16.wgsl, qwen.ts:391-392);
     *  token ids >= vocab give zero rows. */
    embed(tokens, out, M, weight) {
        const name = weight || 'embed';
        const w = this.f16Weights.get(name);
        if (!w) throw new Error(`missing f16 weight: ${name}`);
        const vocab = w.shape[0], C = w.shape[1];
        if (tokens.dtype !== 'u32' || tokens.length < M) throw new Error('embed: tokens must be a u32 tensor of at least M ids');
        if (out.dtype !== 'f32' || out.length < M * C || out.arena !== tokens.arena)
            throw new Error("embed: out must be an f32 [M, C] tensor in the tokens' arena");
        addon.embedF16(this.ctx.handle, this.weights.handle, w.offset, vocab, C, tokens.arena.handle, tokens.offset, M, out.offset);
    }
    /** y = rmsnorm(x (+ residual)) * weight; the sum goes to sumOut (vec_add + rmsnorm.wgsl in one launch). */
    rmsnorm(x, weight, y, M, C, eps, residual, sumOut) {
        const w = this.f32Weights.get(weight);
        if (!w) throw new Error(`missing f32 weight: ${weight}`);
        if (w.length !== C) throw new Error(`rmsnorm: ${weight} has ${w.length} values, C=${C}`);
        for (const t of [y, residual, sumOut]) {
            if (t && t.arena !== x.arena) throw new Error('rmsnorm: x, y, residual and sumOut must share one arena');
        }
        addon.addRmsNorm(this.ctx.handle, x.arena.handle, x.offset, residual ? residual.offset : null,
            this.weights.handle, w.offset, eps, M, C, sumOut ? sumOut.offset : null, y.offset);
    }
    /** out = silu(gate) * up (silu_mul.wgsl, qwen.ts:468-469). */
    siluMul(gate, up, out, n) {
        if (gate.arena !== up.arena || gate.arena !== out.arena) throw new Error('siluMul: tensors must share one arena');
        addon.siluMul(this.ctx.handle, gate.arena.handle, gate.offset, up.offset, n, out.offset);
    }
    /**
     * Cosines and sines of positions 0 .. maxPos - 1 in the weight arena, for KvCache.rotateStore. As an uploaded weight, the table
     * is there when this returns, for any context; a refused one takes no room.
     */
    makeRopeTable(maxPos, rotDim, theta, name) {
        const key = name || 'rope';
        if (this.f32Weights.has(key)) throw new Error(`weight already exists: ${key}`);
        this.ctx.sync();                                       // not during a capture, which would keep the fill for its replays
        const start = this.layout.used;
        const off = this.layout.take(maxPos * rotDim * 4);
        try {
            if (this.layout.used > this.weights.size) throw new Error(`weight arena exhausted (${this.layout.used} > ${this.weights.size})`);
            addon.ropeTable(this.ctx.handle, this.weights.handle, off, maxPos, rotDim, theta);
            this.ctx.sync();
        } catch (e) {
            this.layout.used = start;
            throw e;
        }
        this.f32Weights.set(key, new Tensor(this.weights, off, maxPos * rotDim, [maxPos, rotDim], 'f32'));
    }
    /**
     * Over M rows of V logits: logprobs [M, T] of tokens (i32 [M, T]; -1: none), entropy [M], topIds (i32) and topLogprobs
     * [M, k]; each may be left out (tokens with logprobs, topIds with topLogprobs). T and k are the tensors' second dimension:
     * tensors of more rows serve smaller passes. Tensors of one dimension hold one value a row.
     */
    tokenLogprobs(logits, M, V, o) {
        if (!o.tokens !== !o.logprobs || !o.topIds !== !o.topLogprobs) throw new Error('tokenLogprobs: tokens come with logprobs, topIds with topLogprobs');
        for (const t of [o.tokens, o.logprobs, o.entropy, o.topIds, o.topLogprobs]) {
            if (t && t.arena !== logits.arena) throw new Error('tokenLogprobs: tensors must share one arena');
        }
        const bad = (t, dtype) => t && t.dtype !== dtype;
        if (!(M >= 1) || logits.dtype !== 'f32' || logits.length < M * V || (o.entropy && o.entropy.length < M) ||
            [o.logprobs, o.entropy, o.topLogprobs].some((t) => bad(t, 'f32')) || [o.tokens, o.topIds].some((t) => bad(t, 'i32')))
            throw new Error('tokenLogprobs: a tensor is too small or of another type');
        // values a row of two tensors that belong together
        const width = (t, same) => {
            if (!t) return 0;
            if (t.shape.length !== 2 && !(t.shape.length === 1 && t.length === M))
                throw new Error('tokenLogprobs: tokens and topIds must be [rows, values a row] or [M]');
            const w = t.shape.length === 2 ? t.shape[1] : 1;
            if (t.length < M * w || same.length < M * w || (same.shape.length === 2 && same.shape[1] !== w))
                throw new Error('tokenLogprobs: tokens and logprobs must be [M, T] alike, topIds and topLogprobs [M, k]');
            return w;
        };
        const T = width(o.tokens, o.logprobs), k = width(o.topIds, o.topLogprobs);
        const off = (t) => (t ? t.offset : 0);
        addon.tokenLogprobs(this.ctx.handle, logits.arena.handle, logits.offset, V, M, V, off(o.tokens), T, k, off(o.logprobs),
            o.entropy ? o.entropy.offset : null, off(o.topIds), off(o.topLogprobs));
    }
    /** Several linears on one input in one launch (q/k/v, gate/up; qwen.ts:411-413, :464-465). */
    gemmBatch(A, weights, Cs, M) {
        const descs = weights.map((w) => this.linear(w).desc);
        if (!A.pool || Cs.some((c) => c.pool !== A.pool)) throw new Error('gemmBatch: A and every C must come from one ActivationArena');
        const scratch = A.pool.scratchOffset(addon.planBatch(descs, M));
        addon.linearBatch(this.ctx.handle, descs, this.weights.handle, A.arena.handle,
            descs.map(() => A.offset), A.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32, M,
            Cs.map((c) => c.offset), scratch);
    }
    /**
     * Low-rank adapters of a linear, all of them: a fp16 bits [n, rank, K], b fp16 bits [n, N, rank] (Uint16Array), scale [n] (each one's
     * alpha / rank; left out: 1). Adapters of lower ranks have zeros behind their own.
     */
    uploadLora(weight, a, b, n, rank, scale) {
        if (this.loras.has(weight)) throw new Error(`adapters already exist: ${weight}`);
        const { K, N } = this.linear(weight);
        if (!(n >= 1) || rank < 8 || rank > 128 || rank % 8 || K % 8 || N % 4) throw new Error('lora: rank must be 8..128, a multiple of 8, K a multiple of 8, N of 4');
        if (!(a instanceof Uint16Array) || !(b instanceof Uint16Array) || a.length !== n * rank * K || b.length !== n * rank * N || (scale && scale.length !== n))
            throw new Error(`lora: ${weight} is [${N},${K}], ${n} adapters of rank ${rank} do not fit`);
        const s = scale ? Float32Array.from(scale) : new Float32Array(n).fill(1);
        this.loras.set(weight, { aOff: this._place(a), bOff: this._place(b), scaleOff: this._place(s), K, N, rank, nAdapter: n });
    }
    /**
     * Each C [M, N] += scale * (A . a^T) . b^T of its linear's adapters, by each row's id (i32 [M]; -1: none): after gemm or gemmBatch on the
     * same A (f32 or f16), up to 8 linears (q/k/v, gate/up) in one call.
     */
    loraAdd(A, weights, ids, Cs, M) {
        const loras = weights.map((w) => {
            if (!this.loras.has(w)) throw new Error(`missing adapters: ${w}`);
            return this.loras.get(w);
        });
        if (Cs.length !== loras.length) throw new Error(`loraAdd: ${Cs.length} outputs for ${loras.length} linears`);
        if (ids.dtype !== 'i32' || ids.length < M) throw new Error('loraAdd: ids must be an i32 tensor of at least M');
        if ((A.dtype !== 'f32' && A.dtype !== 'f16') || Cs.some((c) => c.dtype !== 'f32')) throw new Error('loraAdd: A must be f32 or f16, C f32');
        if (ids.arena !== A.arena || Cs.some((c) => c.arena !== A.arena)) throw new Error('loraAdd: tensors must share one arena');
        if (loras.some((l, i) => A.length < M * l.K || Cs[i].length < M * l.N)) throw new Error('loraAdd: tensor too small for [M,K] / [M,N]');
        const offs = Cs.map((c) => c.offset);
        batchAddon().loraAdd(this.ctx.handle, loras, this.weights.handle, A.arena.handle, ids.offset, Cs.map(() => A.offset),
            A.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32, M, offs, offs);
    }
    /** fp16 [N,K] copy, bit-identical to the reference's uploaded f16 weight buffer. */
    unpackF16(name, out) {
        const lin = this.linear(name);
        if (out.dtype !== 'f16' || out.length < lin.N * lin.K) throw new Error('unpackF16: output must be an f16 tensor of N*K elements');
        addon.unpack(this.ctx.handle, lin.desc, this.weights.handle, out.arena.handle, out.offset, false);
    }
    /**
     * fp16 [N,K] copies of many weights at once (the loader's whole weight set,
     * qwen-loader.ts:146-162): names[i] into outs[i], same bits as unpackF16, in a few launches.
     */
    unpackAllF16(names, outs) {
        if (names.length !== outs.length) throw new Error('unpackAllF16: one output tensor per weight');
        const descs = names.map((n, i) => {
            const lin = this.linear(n);
            const out = outs[i];
            if (out.dtype !== 'f16' || out.length < lin.N * lin.K) throw new Error('unpackAllF16: output must be an f16 tensor of N*K elements');
            if (out.arena !== outs[0].arena) throw new Error('unpackAllF16: all outputs must share one arena');
            return lin.desc;
        });
        if (descs.length) addon.unpackBatch(this.ctx.handle, descs, this.weights.handle, outs[0].arena.handle, outs.map((o) => o.offset));
    }
    /** fp32 [N,K] = dequantizeGptqInt4 of the stored tensors (computed on the GPU). */
    dequantize(name) {
        const lin = this.linear(name);
        const tmp = this.ctx.arena(lin.N * lin.K * 4);
        try {
            addon.unpack(this.ctx.handle, lin.desc, this.weights.handle, tmp.handle, 0, true);
            return tmp.read(0, new Float32Array(lin.N * lin.K));
        } finally {
            tmp.release();
        }
    }
    release() { this.weights.release(); }
}

// ------------------------------------------------------------------ qwen-loader.ts

const PROJ = [['qW', 'self_attn.q_proj'], ['kW', 'self_attn.k_proj'], ['vW', 'self_attn.v_proj'],
    ['oW', 'self_attn.o_proj'], ['gateW', 'mlp.gate_proj'], ['upW', 'mlp.up_proj'], ['downW', 'mlp.down_proj']];
const BIASED = new Set(['qW', 'kW', 'vW']);

function qwenLinearShapes(c) {
    const C = c.nEmbd, HI = qwenKvDim(c), I = c.intermediate;
    return { qW: [C, C], kW: [C, HI], vW: [C, HI], oW: [C, C], gateW: [C, I], upW: [C, I], downW: [I, C] };
}

const QWEN_LOCAL_DIR = 'models/qwen2.5-0.5b-int4/';   // qwen-loader.ts:27 (public/models layout)

/** A local path or file:// URL -> path (the reference fetches `url`; this host has no network). */
function urlToPath(url) {
    if (/^file:/i.test(url)) return decodeURIComponent(new URL(url).pathname);
    if (/^[a-z][a-z0-9+.-]*:\/\//i.test(url)) throw new Error(`qwen-loader: cannot load ${url}: only a local path or a file:// URL`);
    return url;
}

/** readF16Rows (qwen-loader.ts:70-93): rows [rowStart, rowStart+rowCount) of an F16 tensor as fp32. */
function readF16Rows(file, name, rowStart, rowCount, rowLength) {
    const entry = requireTensor(file, name);
    if (entry.dtype !== 'F16') throw new Error(`qwen-loader: ${name} expected F16, got ${entry.dtype}`);
    if (entry.shape.length !== 2 || entry.shape[0] * rowLength !== entry.shape[0] * entry.shape[1]) {
        throw new Error(`qwen-loader: ${name} shape ${entry.shape} does not match rowLength=${rowLength}`);
    }
    if (rowStart < 0 || rowCount < 0 || rowStart + rowCount > entry.shape[0]) {
        throw new Error(`qwen-loader: rows [${rowStart}, ${rowStart + rowCount}) outside ${name} [${entry.shape}]`);
    }
    const byteStart = file.dataStart + entry.data_offsets[0] + rowStart * rowLength * 2;
    const view = new DataView(file.buffer.buffer, file.buffer.byteOffset + byteStart, rowCount * rowLength * 2);
    const out = new Float32Array(rowCount * rowLength);
    for (let i = 0; i < out.length; i++) out[i] = f16BitsToF32(view.getUint16(i * 2, true));
    return out;
}

/**
 * desc_act=false: g_idx, when present, must be the identity map i / group (qwen-format.ts:125-130).
 * The fused kernels assume it, so an act-order checkpoint is rejected rather than loaded wrong.
 */
function checkGIdx(file, prefix, inFeatures, group) {
    const name = `${prefix}.g_idx`;
    if (!Object.prototype.hasOwnProperty.call(file.header, name)) return;
    expectTensor(file, name, 'I32', [inFeatures]);
    const b = readTensorBytes(file, name);
    const view = new DataView(b.buffer, b.byteOffset, b.byteLength);
    for (let i = 0; i < inFeatures; i++) {
        const g = view.getInt32(i * 4, true);
        if (g !== Math.floor(i / group)) {
            throw new Error(`qwen-loader: ${name}[${i}] = ${g} is not the identity map i/${group} (desc_act checkpoints are not supported)`);
        }
    }
}

/** Adds the stored qzeros nibbles of a linear's real columns into counts[0..15] (qwen-format.ts:112-123). */
function countStoredZeros(qzeros, groups, outFeatures, counts) {
    const nc = Math.ceil(outFeatures / 8);
    const view = new DataView(qzeros.buffer, qzeros.byteOffset, qzeros.byteLength);
    for (let g = 0; g < groups; g++) {
        for (let n = 0; n < outFeatures; n++) {
            const word = view.getUint32((g * nc + (n >> 3)) * 4, true);
            counts[(word >>> (4 * (n & 7))) & 15]++;
        }
    }
    return counts;
}

/**
 * loadQwenWeights (qwen-loader.ts:102-177) for a QuantLinearModel: async, like the reference
 * (`ctx` is unused, as the reference's `_gpu` is; the model holds its context). options (the
 * reference's QwenLoadOptions, qwen-loader.ts:29-38): url (a local path or file:// URL, default
 * QWEN_LOCAL_DIR + 'model.safetensors'), onProgress(done, total, label), keepLayer,
 * keepEmbedRows {start, rows}; and this host's config, groupSize, and path / buffer (a path or an
 * already-read file instead of url). The int4 tensors go to the GPU packed after the shape checks
 * of qwen-format.ts:72-80 and its g_idx identity check; the result (QwenLoadResult, :40-52) adds
 * storedZeros {nibble: count} over every linear (the format probe's stored-zero set, :112-123).
 */
async function loadQwenWeights(ctx, model, options) {
    const opt = options || {};
    const config = opt.config || QWEN25_05B;
    const group = opt.groupSize || 128;
    let raw = opt.buffer;
    if (!raw) {
        const file = opt.path || urlToPath(opt.url !== undefined ? opt.url : `${QWEN_LOCAL_DIR}model.safetensors`);
        raw = await fs.promises.readFile(file);
    }
    const file = parseSafetensors(raw);
    const C = config.nEmbd;
    let tensorCount = 0;
    const emb = requireTensor(file, 'model.embed_tokens.weight');
    if (emb.shape.join(',') !== `${config.vocabSize},${C}`) {
        throw new Error(`qwen-loader: embed_tokens shape [${emb.shape}], expected [${config.vocabSize},${C}]`);
    }
    if (emb.dtype !== 'F16') throw new Error(`qwen-loader: model.embed_tokens.weight expected F16, got ${emb.dtype}`);
    model.uploadF16Bits('embed', readTensorBytes(file, 'model.embed_tokens.weight'), [config.vocabSize, C]);
    tensorCount += 1;
    const embedRows = opt.keepEmbedRows
        ? readF16Rows(file, 'model.embed_tokens.weight', opt.keepEmbedRows.start, opt.keepEmbedRows.rows, C)
        : undefined;
    model.uploadF32('finalNorm', readTensorF32(file, 'model.norm.weight'));
    tensorCount += 1;
    const shapes = qwenLinearShapes(config);
    const zeros = new Array(16).fill(0);
    let kept;
    for (let i = 0; i < config.nLayer; i++) {
        const p = `model.layers.${i}`;
        model.uploadF32(`L${i}.inNorm`, readTensorF32(file, `${p}.input_layernorm.weight`));
        model.uploadF32(`L${i}.postNorm`, readTensorF32(file, `${p}.post_attention_layernorm.weight`));
        tensorCount += 2;
        const layer = {};
        for (const [key, proj] of PROJ) {
            const [K, N] = shapes[key];
            const pre = `${p}.${proj}`;
            const G = Math.ceil(K / group);
            expectTensor(file, `${pre}.qweight`, 'I32', [Math.ceil(K / 8), N]);
            expectTensor(file, `${pre}.qzeros`, 'I32', [G, Math.ceil(N / 8)]);
            expectTensor(file, `${pre}.scales`, 'F16', [G, N]);
            checkGIdx(file, pre, K, group);
            const qzeros = readTensorBytes(file, `${pre}.qzeros`);
            countStoredZeros(qzeros, G, N, zeros);
            const bias = BIASED.has(key) ? readTensorF32(file, `${pre}.bias`) : null;
            model.uploadGptqLinear(`L${i}.${key}`, {
                qweight: readTensorBytes(file, `${pre}.qweight`), qzeros,
                scalesF16: readTensorBytes(file, `${pre}.scales`), inFeatures: K, outFeatures: N,
                groupSize: group, bias,
            });
            tensorCount += bias ? 2 : 1;
            if (opt.keepLayer === i) layer[key] = model.dequantize(`L${i}.${key}`);
        }
        if (opt.keepLayer === i) kept = layer;
        if (opt.onProgress) opt.onProgress(i + 1, config.nLayer, `layer ${i + 1}/${config.nLayer}`);
    }
    const storedZeros = {};
    zeros.forEach((c, v) => { if (c) storedZeros[v] = c; });
    return { gpuBytes: model.weightBytes, tensorCount, fileBytes: raw.byteLength, layer: kept, embedRows, storedZeros };
}

/** {masks: BigUint64Array [M, ceil(M/64)], depths: Int32Array} of a drafted tree: parents[m] is -1 or an earlier row. */
function treeMasks(parents) {
    const list = Array.from(parents), M = list.length;
    list.forEach((p, m) => {                                  // before an Int32Array wraps or rounds them
        if (!Number.isInteger(p) || p < -1 || p >= m) throw libError('QL_E_INVALID', `the parent of row ${m} must be -1 or an earlier row (got ${p})`);
    });
    const masks = new BigUint64Array(M * Math.ceil(M / 64)), depths = new Int32Array(M);
    addon.treeMasks(Int32Array.from(list), masks, depths);
    return { masks, depths };
}

/**
 * Per-layer K and V caches [blockSize, nKvHead * headDim] and the attention over them:
 * QwenGpt's kCache/vCache (qwen.ts:140-141, :200-205), kv_store (:427-428), attention_gqa_cache (:429-440).
 * dtype 'f32', or 'f16' (rotateStore and attendTree only). A pass over drafted tokens (treeMasks) runs rotateStore and
 * attendTree per layer; accept keeps the accepted path.
 */
class KvCache {
    constructor(ctx, config, dtype) {
        this.ctx = ctx;
        this.config = config;
        this.dtype = dtype || 'f32';
        if (this.dtype !== 'f32' && this.dtype !== 'f16') throw new Error(`kv cache: dtype ${dtype}`);
        this.D = qwenHeadDim(config);
        this.rowLen = qwenKvDim(config);
        this.rowBytes = this.rowLen * (this.dtype === 'f16' ? 2 : 4);
        this.region = Math.ceil(config.blockSize * this.rowBytes / 256) * 256;
        this.arena = ctx.arena(2 * config.nLayer * this.region);
        this.regions = Array.from({ length: 2 * config.nLayer }, (_, i) => i * this.region);
    }
    offsets(layer) {
        if (layer < 0 || layer >= this.config.nLayer) throw new Error(`layer ${layer} out of range`);
        return [2 * layer * this.region, (2 * layer + 1) * this.region];
    }
    _f32Only(what) {
        if (this.dtype !== 'f32') throw new Error(`${what}: an fp16 cache takes rotateStore and attendTree`);
    }
    store(layer, k, v, rows, pos0) {
        this._f32Only('store');
        const [ko, vo] = this.offsets(layer);
        if (k.arena !== v.arena) throw new Error('store: k and v must share one arena');
        addon.kvStore(this.ctx.handle, k.arena.handle, k.offset, this.arena.handle, ko, this.config.blockSize, rows, this.rowLen, pos0);
        addon.kvStore(this.ctx.handle, v.arena.handle, v.offset, this.arena.handle, vo, this.config.blockSize, rows, this.rowLen, pos0);
    }
    attend(layer, q, out, M, pastLen) {
        this._f32Only('attend');
        const c = this.config;
        if (q.arena !== out.arena) throw new Error('attend: q and out must share one arena');
        const [ko, vo] = this.offsets(layer);
        addon.attention(this.ctx.handle, q.arena.handle, q.offset, this.arena.handle, ko, vo, c.blockSize, M,
            c.nHead, c.nKvHead, this.D, pastLen, out.offset);
    }
    /**
     * q and k turned by positions (i32 [M]) and normed per head where weights are named; q to qOut, k and v to rows slot0 + m. A row
     * whose position the table does not have is padding: its qOut and cache rows stay as they were (qOut = q: unturned), so the
     * table needs as many positions as the text may have.
     */
    rotateStore(layer, model, q, k, v, positions, qOut, M, slot0, options) {
        const o = options || {}, c = this.config;
        if ([k, v, positions, qOut].some((t) => t.arena !== q.arena)) throw new Error('rotateStore: tensors must share one arena');
        if (q.length < M * c.nHead * this.D || qOut.length < M * c.nHead * this.D || k.length < M * this.rowLen || v.length < M * this.rowLen ||
            [q, k, v, qOut].some((t) => t.dtype !== 'f32') || positions.dtype !== 'i32' || positions.length < M)
            throw new Error('rotateStore: a tensor is too small or of another type');
        const weight = (name, length) => {
            const w = model.f32Weights.get(name);
            if (!w || (length ? w.length !== length : w.shape.length !== 2)) throw new Error(`missing f32 weight: ${name}`);
            return w;
        };
        const table = weight(o.rope || 'rope');
        const [ko, vo] = this.offsets(layer);
        addon.qkNormRope(this.ctx.handle, {
            tableOff: table.offset, maxPos: table.shape[0], nHead: c.nHead, nKvHead: c.nKvHead, D: this.D, rotDim: table.shape[1], interleaved: 0,
            qNormOff: o.qNorm ? weight(o.qNorm, this.D).offset : null, kNormOff: o.kNorm ? weight(o.kNorm, this.D).offset : null,
            normEps: o.eps === undefined ? 1e-6 : o.eps, qStride: 0, kStride: 0, vStride: 0, cacheDtype: this.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32,
        }, model.weights.handle, q.arena.handle, q.offset, k.offset, v.offset, positions.offset, M, qOut.offset, this.arena.handle, ko, vo,
        c.blockSize, slot0);
    }
    /** GQA attention of M <= 256 drafted rows at pastLen + m; masks: a u64 tensor of treeMasks' words, or null for causal rows. */
    attendTree(layer, q, out, M, pastLen, masks) {
        const c = this.config;
        if (q.arena !== out.arena || (masks && masks.arena !== q.arena)) throw new Error('attendTree: q, out and masks must share one arena');
        if (q.dtype !== 'f32' || out.dtype !== 'f32' || q.length < M * c.nHead * this.D || out.length < M * c.nHead * this.D ||
            (masks && (masks.dtype !== 'u64' || masks.length < M * Math.ceil(M / 64))))
            throw new Error('attendTree: a tensor is too small or of another type');
        const [ko, vo] = this.offsets(layer);
        addon.attentionTree(this.ctx.handle, q.arena.handle, q.offset, this.arena.handle, ko, vo, this.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32,
            c.blockSize, M, c.nHead, c.nKvHead, this.D, pastLen, masks ? masks.offset : null, out.offset);
    }
    /** Row pastLen + i of every layer becomes row pastLen + path[i] (i32, i < n): an accepted path of the tree at pastLen. */
    accept(pastLen, path, n) {
        if (path.dtype !== 'i32' || path.length < n) throw new Error('accept: path must be an i32 tensor of at least n rows');
        const T = this.config.blockSize;
        addon.kvMove(this.ctx.handle, this.arena.handle, this.regions, T, this.arena.handle, this.regions, T, this.rowBytes, pastLen, pastLen, n,
            path.arena.handle, path.offset);
    }
    /**
     * The first rows of every layer into another cache of the same layers, heads and dtype. A cache of another context: the copy
     * runs on this one's stream, and the host waits for the other stream before it and for the copy after it.
     */
    fork(to, rows) {
        if (to.config.nLayer !== this.config.nLayer || to.config.nKvHead !== this.config.nKvHead || to.D !== this.D || to.dtype !== this.dtype)
            throw new Error('fork: the caches differ in layers, heads or dtype');
        const apart = to.ctx !== this.ctx;
        if (apart) { this.ctx.sync(); to.ctx.sync(); }
        addon.kvMove(this.ctx.handle, to.arena.handle, to.regions, to.config.blockSize, this.arena.handle, this.regions, this.config.blockSize,
            this.rowBytes, 0, 0, rows, null, null);
        if (apart) this.ctx.sync();
    }
    release() { this.arena.release(); }
}

/**
 * K and V of many sequences in pages that they take as they grow, in one device arena, for passes over many requests at once: append and
 * attend run per layer over a batch. dtype 'f16', or 'f8': e4m3 values with a power of two for every 16 tokens of a head. Sequences are
 * numbers (newSequence); what they hold is counted on the host. batch() takes the pages that a pass needs and counts its tokens, so it is
 * called once, before the pass's layers; its tables are read on the device when a pass runs.
 */
class PagedKvCache {
    constructor(ctx, config, pages, pageSize, dtype) {
        this.dtype = dtype || 'f16';
        this.pageSize = pageSize || 64;
        if (this.dtype !== 'f16' && this.dtype !== 'f8') throw new Error(`paged kv cache: dtype ${dtype}`);
        if (!(pages >= 1) || ![64, 128, 256].includes(this.pageSize)) throw new Error('paged kv cache: at least one page, of 64, 128 or 256 tokens');
        this.ctx = ctx;
        this.config = config;
        this.pages = pages;
        this.D = qwenHeadDim(config);
        this.rowLen = qwenKvDim(config);
        if (this.D < 16 || this.D > 256 || this.D % 16 || config.nHead > 4096 || config.nHead % config.nKvHead)
            throw new Error('paged kv cache: head dim must be 16..256, a multiple of 16, nHead at most 4096, a multiple of nKvHead');
        const f8 = this.dtype === 'f8';
        this.pageBytes = this.pageSize * this.rowLen * (f8 ? 1 : 2);
        this.scaleBytes = f8 ? config.nKvHead * (this.pageSize / 16) * 4 : 0;      // of a page
        const layout = new ArenaLayout();
        this.regions = Array.from({ length: 2 * config.nLayer }, () => layout.take(pages * this.pageBytes));
        this.scales = f8 ? Array.from({ length: 2 * config.nLayer }, () => layout.take(pages * this.scaleBytes)) : [];
        this.arena = ctx.arena(layout.used);
        this._free = Array.from({ length: pages }, (_, i) => pages - 1 - i);
        this._users = new Array(pages).fill(0);           // sequences that hold a page
        this._lists = new Map();
        this._lengths = new Map();
        this._next = 0;
    }
    get freePages() { return this._free.length; }
    newSequence() {
        const s = this._next++;
        this._lists.set(s, []);
        this._lengths.set(s, 0);
        return s;
    }
    length(sequence) { return this._lengths.get(this._known(sequence)); }
    _known(sequence) {
        if (!this._lists.has(sequence)) throw new Error(`no such sequence: ${sequence}`);
        return sequence;
    }
    _take() {
        const p = this._free.pop();
        this._users[p] = 1;
        return p;
    }
    _drop(page) { if (--this._users[page] === 0) this._free.push(page); }
    _copy(page) {
        const to = this._take();
        for (const [offs, size] of [[this.regions, this.pageBytes], [this.scales, this.scaleBytes]]) {
            for (let i = 0; i < offs.length; i += 256) {
                const some = offs.slice(i, i + 256);
                addon.kvMove(this.ctx.handle, this.arena.handle, some, this.pages, this.arena.handle, some, this.pages, size, to, page, 1, null, null);
            }
        }
        return to;
    }
    /** A finished sequence's pages go back, but for those that others hold. */
    free(sequence) {
        for (const p of this._lists.get(this._known(sequence))) this._drop(p);
        this._lists.delete(sequence);
        this._lengths.delete(sequence);
    }
    /** The sequence's first tokens are kept (a rejected draft, an edited prompt). */
    cut(sequence, tokens) {
        if (!(tokens >= 0 && tokens <= this.length(sequence)) || !Number.isInteger(tokens)) throw new Error(`cut: sequence ${sequence} has ${this.length(sequence)} tokens`);
        const pages = this._lists.get(sequence);
        while (pages.length > Math.ceil(tokens / this.pageSize)) this._drop(pages.pop());
        this._lengths.set(sequence, tokens);
    }
    /** A sequence that continues another one: its whole pages are shared, the last one, where it is not full, is copied. */
    fork(sequence) {
        const tokens = this.length(sequence), pages = this._lists.get(sequence), whole = Math.floor(tokens / this.pageSize);
        if (whole < pages.length && !this._free.length) throw new Error('fork: no page left');
        const s = this.newSequence(), own = pages.slice(0, whole);
        for (const p of own) this._users[p]++;
        this._lists.set(s, own);
        this._lengths.set(s, tokens);
        if (whole < pages.length) own.push(this._copy(pages[whole]));
        return s;
    }
    /**
     * Rows of a pass: [sequence, rows] in the order of the rows, each sequence once. Takes the pages that their tokens need and counts the tokens;
     * M: rows of the pass's tensors (those behind the sequences' are padding). A batch that is refused takes nothing. After a pass that fails later (a
     * rope table of fewer positions, for one) its sequences are cut back to their earlier lengths: the tokens counted are in no page.
     */
    batch(pool, sequences, M) {
        const order = sequences.map(([s]) => this._known(s)), rows = sequences.map(([, n]) => n);
        if (!order.length || new Set(order).size !== order.length || rows.some((n) => !Number.isInteger(n) || n < 0))
            throw new Error('batch: at least one sequence, each once, with no negative rows');
        const total = rows.reduce((a, b) => a + b, 0), m = M === undefined ? Math.max(total, 1) : M, P = this.pageSize;
        if (m < total) throw new Error(`batch: ${total} rows for tensors of ${m}`);
        const lists = order.map((s) => this._lists.get(s)), lengths = order.map((s, i) => this._lengths.get(s) + rows[i]);
        const longest = lengths.reduce((x, y) => Math.max(x, y)), { nHead, nKvHead } = this.config;
        if (!(m >= 1 && m <= BATCH.rows) || !Number.isInteger(m) || order.length > BATCH.seqs || longest > BATCH.tokens)
            throw new Error(`batch: 1 to ${BATCH.rows} rows, at most ${BATCH.seqs} sequences, ${BATCH.tokens} tokens of one (got ${m}, ${order.length}, ${longest})`);
        if (m * (nHead + 2 * nKvHead) > BATCH.heads || order.length * nKvHead > BATCH.seqHeads)
            throw new Error(`batch: more than ${BATCH.heads} heads of rows or ${BATCH.seqHeads} kv heads of sequences`);
        // a page that the pass appends to is the sequence's alone: one that others hold as well (cut in the middle of a shared one) is copied first,
        // by all who append to it, or by all but the last where nobody else holds it
        const at = order.map((s, i) => (rows[i] && this._lengths.get(s) % P ? Math.floor(this._lengths.get(s) / P) : -1));
        const writers = new Map();
        at.forEach((k, i) => { if (k >= 0) writers.set(lists[i][k], (writers.get(lists[i][k]) || 0) + 1); });
        let need = 0;
        for (const [p, n] of writers) need += n - (this._users[p] === n ? 1 : 0);
        lengths.forEach((L, i) => { need += Math.max(0, Math.ceil(L / P) - lists[i].length); });
        if (need > this._free.length) throw new Error(`batch: ${need} pages for ${this._free.length} that are left`);
        const most = Math.max(1, ...lengths.map((L, i) => Math.max(lists[i].length, Math.ceil(L / P))));
        const rowStart = pool.alloc([order.length + 1], 'i32'), kvLen = pool.alloc([order.length], 'i32'), pages = pool.alloc([order.length, most], 'i32');
        at.forEach((k, i) => {
            if (k < 0 || this._users[lists[i][k]] === 1) return;
            const to = this._copy(lists[i][k]);
            this._drop(lists[i][k]);
            lists[i][k] = to;
        });
        const table = new Int32Array(order.length * most).fill(-1), starts = new Int32Array(order.length + 1);
        order.forEach((s, i) => {
            while (lists[i].length < Math.ceil(lengths[i] / P)) lists[i].push(this._take());
            this._lengths.set(s, lengths[i]);
            table.set(lists[i], i * most);
            starts[i + 1] = starts[i] + rows[i];
        });
        rowStart.write(starts);
        kvLen.write(Int32Array.from(lengths));
        pages.write(table);
        const desc = {
            rowStartOff: rowStart.offset, kvLenOff: kvLen.offset, pagesOff: pages.offset, nSeq: order.length, maxPages: most,
            maxRows: Math.max(1, ...rows), maxLen: Math.max(1, ...lengths),
        };
        return { desc, M: m, rows: total, tables: [rowStart, kvLen, pages] };
    }
    desc(layer) {
        if (!(layer >= 0 && layer < this.config.nLayer)) throw new Error(`layer ${layer} out of range`);
        const k = 2 * layer, v = k + 1, f8 = this.dtype === 'f8';
        return {
            kOff: this.regions[k], vOff: this.regions[v], kScaleOff: f8 ? this.scales[k] : null, vScaleOff: f8 ? this.scales[v] : null, nPage: this.pages,
            pageSize: this.pageSize, nKvHead: this.config.nKvHead, D: this.D, cacheDtype: f8 ? QL_DTYPE_F8 : QL_DTYPE_F16,
        };
    }
    /**
     * q and k turned by their rows' positions, normed per head first where weights are named; q to qOut (f32, where q itself may be given, or f16),
     * k and v to their places in the sequences' pages. Rows of padding stay as they were.
     */
    append(layer, model, q, k, v, batch, qOut, options) {
        const o = options || {}, c = this.config, M = batch.M;
        if ([k, v, qOut, ...batch.tables].some((t) => t.arena !== q.arena)) throw new Error('append: tensors must share one arena');
        if (q.length < M * c.nHead * this.D || qOut.length < M * c.nHead * this.D || k.length < M * this.rowLen || v.length < M * this.rowLen ||
            [q, k, v].some((t) => t.dtype !== 'f32') || (qOut.dtype !== 'f32' && qOut.dtype !== 'f16'))
            throw new Error('append: a tensor is too small or of another type');
        const weight = (name, length) => {
            const w = model.f32Weights.get(name);
            if (!w || (length ? w.length !== length : w.shape.length !== 2)) throw new Error(`missing f32 weight: ${name}`);
            return w;
        };
        const table = weight(o.rope || 'rope'), paged = this.desc(layer);
        batchAddon().pagedAppend(this.ctx.handle, {
            tableOff: table.offset, maxPos: table.shape[0], nHead: c.nHead, nKvHead: c.nKvHead, D: this.D, rotDim: table.shape[1], interleaved: 0,
            qNormOff: o.qNorm ? weight(o.qNorm, this.D).offset : null, kNormOff: o.kNorm ? weight(o.kNorm, this.D).offset : null,
            normEps: o.eps === undefined ? 1e-6 : o.eps, qStride: 0, kStride: 0, vStride: 0, cacheDtype: paged.cacheDtype,
        }, model.weights.handle, q.arena.handle, q.offset, k.offset, v.offset, batch.desc, M, qOut.offset,
        qOut.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32, this.arena.handle, paged);
    }
    /** out [M, nHead * D] = causal GQA attention of the batch's rows over their sequences; q and out both f32 or both f16. */
    attend(layer, q, out, batch) {
        const c = this.config, M = batch.M;
        if ([out, ...batch.tables].some((t) => t.arena !== q.arena)) throw new Error('attend: q, out and the batch must share one arena');
        if ((q.dtype !== 'f32' && q.dtype !== 'f16') || out.dtype !== q.dtype || q.length < M * c.nHead * this.D || out.length < M * c.nHead * this.D)
            throw new Error('attend: a tensor is too small or of another type');
        batchAddon().pagedAttention(this.ctx.handle, q.arena.handle, q.offset, q.dtype === 'f16' ? QL_DTYPE_F16 : QL_DTYPE_F32, this.arena.handle,
            this.desc(layer), batch.desc, M, c.nHead, out.offset);
    }
    release() { this.arena.release(); }
}

module.exports = {
    addon, ADDON_PATH, QL_DTYPE_F32, QL_DTYPE_F16, QWEN25_05B, qwenHeadDim, qwenKvDim, Seq,
    dtypeByteSize, parseSafetensorsHeader, parseSafetensors, tensorCount, requireTensor,
    expectTensor, f16BitsToF32, readTensorBytes, readTensorF32, ArenaLayout, Arena, Context,
    makeDesc, dequantizeGptqInt4, Tensor, ActivationArena, QuantLinearModel,
    qwenLinearShapes, loadQwenWeights, KvCache, QWEN_LOCAL_DIR, urlToPath, readF16Rows, checkGIdx,
    countStoredZeros, treeMasks, get batchAddon() { return batchAddon(); }, QL_DTYPE_F8, PagedKvCache,
};
