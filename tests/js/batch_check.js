'use strict';
/**
 * Drives the Node host's passes over many requests for tests/test_batch_node.py; prints one JSON line.
 *
 *   node batch_check.js host        no GPU: the addon's functions, pages of sequences, refusals
 *   node batch_check.js gpu <dir>   passes over several sequences with adapters: files of <dir> in, files out (cases.json)
 */
const fs = require('fs');
const path = require('path');
const q = require('../../webllm_amd/js');

function message(fn) {
    try { fn(); return null; } catch (e) { return e.message; }
}

function host() {
    const config = { nLayer: 2, nHead: 6, nKvHead: 2, nEmbd: 384 };
    const written = new Map();
    const ctx = { handle: {}, arena: (size) => ({ handle: {}, size, write: (off, t) => written.set(off, Array.from(t)) }) };
    const kv = new q.PagedKvCache(ctx, config, 6, 64, 'f8'), pool = new q.ActivationArena(ctx, 1 << 20);
    const tables = (b) => b.tables.map((t) => written.get(t.offset));
    const a = kv.newSequence(), b = kv.newSequence();
    const first = kv.batch(pool, [[a, 70], [b, 1]], 80);
    const one = { desc: first.desc, M: first.M, rows: first.rows, tables: tables(first), free: kv.freePages };
    const refused = [() => kv.batch(pool, []), () => kv.batch(pool, [[a, 1], [a, 1]]), () => kv.batch(pool, [[a, -1]]), () => kv.batch(pool, [[a, 0.5]]), () => kv.batch(pool, [[9, 1]]),
        () => kv.batch(pool, [[a, 5]], 4), () => kv.batch(pool, [[a, 59 + 64 * 4]]), () => kv.cut(a, 71), () => kv.cut(a, 1.5), () => kv.length(7), () => kv.free(7), () => kv.desc(2),
        () => new q.PagedKvCache(ctx, config, 0), () => new q.PagedKvCache(ctx, config, 4, 32), () => new q.PagedKvCache(ctx, config, 4, 64, 'f32')].map(message);
    const kept = [kv.length(a), kv.length(b), kv.freePages];
    kv.batch(pool, [[b, 127], [a, 0]]);
    const c = kv.fork(b);                                      // whole pages: shared
    const shared = [kv.freePages, kv.length(c), kv._lists.get(c).join() === kv._lists.get(b).join()];
    kv.free(b);
    const after = [kv.freePages];
    kv.free(c);
    kv.cut(a, 64);
    after.push(kv.freePages);
    const desc = kv.desc(1);
    const T = (shape, dtype, arena) => new q.Tensor(arena || pool.arena, 0, shape.reduce((x, y) => x * y, 1), shape, dtype || 'f32');
    const batch = kv.batch(pool, [[a, 6]]);
    const model = Object.assign(Object.create(q.QuantLinearModel.prototype), {
        ctx, weights: { handle: {} }, f32Weights: new Map([['rope', T([256, 64])], ['n', T([32])]]), linears: new Map([['w', { K: 64, N: 32 }]]), loras: new Map(), _place: () => 0,
    });
    const Q = T([6, 384]), K = T([6, 128]), O = T([6, 384]), H = T([6, 384], 'f16'), KH = T([6, 128], 'f16'), S = T([5, 384]), F = T([6, 384], 'f32', {});
    const calls = [() => kv.append(0, model, Q, K, KH, batch, O), () => kv.append(0, model, H, K, K, batch, O), () => kv.append(0, model, S, K, K, batch, O), () => kv.append(0, model, Q, K, K, batch, F),
        () => kv.append(0, model, Q, K, K, batch, O, { rope: 'x' }), () => kv.append(0, model, Q, K, K, batch, O, { qNorm: 'n' }), () => kv.attend(0, Q, H, batch), () => kv.attend(0, S, O, batch),
        () => kv.attend(0, Q, F, batch), () => kv.attend(2, Q, O, batch)].map(message);
    const A = new Uint16Array(3 * 8 * 64), B = new Uint16Array(3 * 8 * 32);
    const lora = [() => model.uploadLora('w', A.subarray(1), B, 3, 8), () => model.uploadLora('w', A, B, 3, 8, [1, 2]), () => model.uploadLora('w', A, B, 2, 12), () => model.uploadLora('x', A, B, 3, 8),
        () => model.uploadLora('w', Float32Array.from(A), B, 3, 8)].map(message);
    model.uploadLora('w', A, B, 3, 8);
    const X = T([6, 64]), C = T([6, 32]), I = T([6], 'i32');
    lora.push(...[() => model.uploadLora('w', A, B, 3, 8), () => model.loraAdd(X, ['v'], I, [C], 6), () => model.loraAdd(X, ['w'], I, [C, C], 6), () => model.loraAdd(X, ['w'], C, [C], 6),
        () => model.loraAdd(X, ['w'], I, [T([6, 32], 'f16')], 6), () => model.loraAdd(X, ['w'], I, [C], 7), () => model.loraAdd(F, ['w'], I, [C], 6)].map(message));
    const library = [() => kv.append(0, model, Q, K, K, batch, H), () => kv.attend(0, H, H, batch), () => model.loraAdd(X, ['w'], I, [C], 6), () => q.batchAddon.loraAdd(1, 2)].map(message);
    console.log(JSON.stringify({ functions: Object.getOwnPropertyNames(q.batchAddon).filter((n) => typeof q.batchAddon[n] === 'function').sort(), one, refused, kept, shared, after, desc, calls, lora, library }));
}

function gpu(dir) {
    const c = JSON.parse(fs.readFileSync(path.join(dir, 'cases.json'), 'utf8'));
    const bytes = (f) => Uint8Array.from(fs.readFileSync(path.join(dir, f)));
    const ctx = new q.Context(0);
    const cfg = c.config;
    const model = new q.QuantLinearModel(ctx, 4 << 20);
    model.makeRopeTable(256, cfg.nEmbd / cfg.nHead, cfg.ropeTheta);
    model.uploadF32('qn', c.qn);
    model.uploadGptqLinear('w', { qweight: new Uint8Array(cfg.nEmbd * 128 / 2), qzeros: null, scalesF16: new Uint16Array(cfg.nEmbd), inFeatures: cfg.nEmbd, outFeatures: 128 });
    model.uploadLora('w', new Uint16Array(bytes('A').buffer), new Uint16Array(bytes('B').buffer), 3, 8, c.scale);
    const pool = new q.ActivationArena(ctx, 8 << 20);
    for (const dtype of ['f16', 'f8']) {
        const kv = new q.PagedKvCache(ctx, cfg, 12, 64, dtype);
        const seqs = [kv.newSequence(), kv.newSequence()];
        c.passes.forEach((p, i) => {
            if (p.fork !== undefined) seqs.push(kv.fork(seqs[p.fork]));
            if (p.cut) kv.cut(seqs[p.cut[0]], p.cut[1]);
            const batch = kv.batch(pool, p.rows.map(([s, n]) => [seqs[s], n]), p.M), M = batch.M;
            const T = (n, shape, dt) => { const t = pool.alloc(shape, dt); t.write(bytes(`${n}${i}`)); return t; };
            const Q = T('q', [M, cfg.nEmbd]), K = T('k', [M, kv.rowLen]), V = T('v', [M, kv.rowLen]), I = T('ids', [M], 'i32');
            const O = pool.alloc([M, cfg.nEmbd]), Y = T('v', [M, 128]);
            O.write(new Float32Array(M * cfg.nEmbd));
            kv.append(1, model, Q, K, V, batch, Q, { qNorm: 'qn' });
            kv.attend(1, Q, O, batch);
            model.loraAdd(O, ['w'], I, [Y], M);
            for (const [n, t] of [['o', O], ['y', Y]]) {
                const r = t.read();
                fs.writeFileSync(path.join(dir, `${n}${i}.${dtype}`), Buffer.from(r.buffer, r.byteOffset, r.byteLength));
            }
            pool.reset();
        });
        kv.release();
    }
    pool.release();
    model.release();
    ctx.destroy();
    console.log('{}');
}

const [mode, dir] = process.argv.slice(2);
if (mode === 'host') host();
else gpu(dir);
