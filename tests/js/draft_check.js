'use strict';
/**
 * Drives the Node host's speculative decoding for tests/test_draft.py.
 *
 *   node draft_check.js abi         no GPU: the addon's functions, masks of trees, refusals; prints one JSON line
 *   node draft_check.js gpu <dir>   one drafted pass over a cache: files of <dir> in, files out (cases.json)
 */
const fs = require('fs');
const path = require('path');
const q = require('../../webllm_amd/js');

function message(fn) {
    try { fn(); return null; } catch (e) { return e.message; }
}

function abi() {
    const names = ['ropeTable', 'qkNormRope', 'treeMasks', 'attentionTree', 'tokenLogprobs', 'kvMove'];
    const parents = Array.from({ length: 70 }, (_, m) => (m === 0 ? -1 : Math.floor(m / 2) - (m % 3 === 0 ? 1 : 0)));
    const r = q.treeMasks(parents);
    console.log(JSON.stringify({
        functions: names.filter((n) => typeof q.addon[n] === 'function'), parents,
        masks: Array.from(r.masks, String), depths: Array.from(r.depths),
        bad: message(() => q.treeMasks([0])), short: message(() => q.addon.treeMasks(new Int32Array(3), new BigUint64Array(2), new Int32Array(3))),
        few: message(() => q.addon.attentionTree(1, 2)), noHandle: message(() => q.addon.ropeTable({}, {}, 0, 1, 8, 1e4)),
    }));
}

function gpu(dir) {
    const c = JSON.parse(fs.readFileSync(path.join(dir, 'cases.json'), 'utf8'));
    const bytes = (f) => Uint8Array.from(fs.readFileSync(path.join(dir, f)));
    const out = (f, t) => fs.writeFileSync(path.join(dir, f), Buffer.from(t.buffer, t.byteOffset, t.byteLength));
    const ctx = new q.Context(0);
    const cfg = c.config, M = c.M, D = cfg.nEmbd / cfg.nHead;
    const model = new q.QuantLinearModel(ctx, 4 << 20);
    model.makeRopeTable(cfg.blockSize, D, cfg.ropeTheta);
    model.uploadF32('qn', c.qn);
    const pool = new q.ActivationArena(ctx, 8 << 20);
    const errors = {};
    for (const dtype of ['f32', 'f16']) {
        const kv = new q.KvCache(ctx, cfg, dtype);
        const other = new q.KvCache(ctx, cfg, dtype);
        const T = (n, shape, dt) => { const t = pool.alloc(shape, dt); t.write(bytes(n)); return t; };
        // the context, causal, then the tree
        {
            const Q = T('q0', [c.past, cfg.nEmbd]), K = T('k0', [c.past, kv.rowLen]), V = T('v0', [c.past, kv.rowLen]);
            const pos = T('pos0', [c.past], 'i32');
            kv.rotateStore(1, model, Q, K, V, pos, Q, c.past, 0, { qNorm: 'qn' });
        }
        const Q = T('q1', [M, cfg.nEmbd]), K = T('k1', [M, kv.rowLen]), V = T('v1', [M, kv.rowLen]), pos = T('pos1', [M], 'i32');
        const { masks, depths } = q.treeMasks(c.parents);
        const W = pool.alloc([masks.length], 'u64');
        W.write(masks);
        const O = pool.alloc([M, cfg.nEmbd]), QR = pool.alloc([M, cfg.nEmbd]);
        kv.rotateStore(1, model, Q, K, V, pos, QR, M, c.past, { qNorm: 'qn' });
        kv.attendTree(1, QR, O, M, c.past, W);
        const X = T('x', [M, c.V]), tok = T('tok', [M, 2], 'i32');
        const lp = pool.alloc([M, 2]), ent = pool.alloc([M]), ids = pool.alloc([M, 3], 'i32'), tlp = pool.alloc([M, 3]);
        model.tokenLogprobs(X, M, c.V, { tokens: tok, logprobs: lp, entropy: ent, topIds: ids, topLogprobs: tlp });
        const P = T('path', [c.path], 'i32');
        kv.accept(c.past, P, c.path);
        kv.fork(other, c.past + c.path);
        // one more token after the accepted path, over the forked cache
        const Q2 = T('q2', [1, cfg.nEmbd]), K2 = T('k2', [1, kv.rowLen]), V2 = T('v2', [1, kv.rowLen]), p2 = T('pos2', [1], 'i32');
        const O2 = pool.alloc([1, cfg.nEmbd]);
        other.rotateStore(1, model, Q2, K2, V2, p2, Q2, 1, c.past + c.path, { qNorm: 'qn' });
        other.attendTree(1, Q2, O2, 1, c.past + c.path);
        ctx.sync();
        for (const [n, t] of [['o', O], ['o2', O2], ['lp', lp], ['ent', ent], ['ids', ids], ['tlp', tlp]]) out(`${n}.${dtype}`, t.read());
        if (Array.from(depths).join() !== c.depths.join()) throw new Error('depths');
        errors.store = message(() => { if (dtype === 'f16') kv.store(0, K, V, 1, 0); });
        errors.attend = message(() => { if (dtype === 'f16') kv.attend(0, Q, O, 1, 0); });
        errors.type = message(() => kv.attendTree(0, Q, O, M, 0, pos));
        errors.range = message(() => kv.attendTree(0, Q, O, M, cfg.blockSize, W));
        errors.path = message(() => kv.accept(0, P, c.path + 1));
        errors.missing = message(() => kv.rotateStore(1, model, Q, K, V, pos, QR, M, 0, { kNorm: 'nothing' }));
        errors.pair = message(() => model.tokenLogprobs(X, M, c.V, { tokens: tok }));
        const H = pool.alloc([M, cfg.nEmbd], 'f16');
        errors.half = message(() => kv.attendTree(0, H, O, M, 0, W));
        errors.halfOut = message(() => kv.rotateStore(1, model, Q, K, V, pos, H, M, 0));
        errors.regions = message(() => q.addon.kvMove(ctx.handle, kv.arena.handle, [0, kv.region], cfg.blockSize, other.arena.handle, [0], cfg.blockSize,
            kv.rowBytes, 0, 0, 1, null, null));
        kv.release();
        other.release();
        pool.reset();
    }
    errors.dtype = message(() => new q.KvCache(ctx, cfg, 'bf16'));
    pool.release();
    model.release();
    ctx.destroy();
    console.log(JSON.stringify({ errors }));
}

const [mode, dir] = process.argv.slice(2);
if (mode === 'abi') abi();
else gpu(dir);
