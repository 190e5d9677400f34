'use strict';
/**
 * Drives the Node host's speculative decoding for tests/test_draft_hosts.py; prints one JSON line.
 *
 *   node draft_hosts_check.js widths   no GPU: tensors of log probabilities that are taken and refused
 *   node draft_hosts_check.js fork     no GPU: which contexts a fork waits for
 *   node draft_hosts_check.js trees    no GPU: parents of drafted trees
 *   node draft_hosts_check.js table    no GPU: rope tables that are refused
 *   node draft_hosts_check.js read     no GPU: arrays that tensors read into
 *   node draft_hosts_check.js exports  no GPU: the addon's functions
 *   node draft_hosts_check.js gpu      log probabilities into buffers of more rows than the pass has
 */
const q = require('../../webllm_amd/js');

function message(fn) {
    try { fn(); return null; } catch (e) { return e.message; }
}

const arena = { handle: {} };
const tensor = (shape, dtype) => new q.Tensor(arena, 0, shape.reduce((a, b) => a * b, 1), shape, dtype || 'f32');

function widths() {
    const model = Object.assign(Object.create(q.QuantLinearModel.prototype), { ctx: { handle: {} } });
    const x = tensor([256, 100]), ent = tensor([256]);
    const call = (M, o) => message(() => model.tokenLogprobs(x, M, 100, o));
    const pair = (a, b) => ({ tokens: tensor(a, 'i32'), logprobs: tensor(b) });
    const top = (a, b) => ({ topIds: tensor(a, 'i32'), topLogprobs: tensor(b) });
    return {
        taken: [call(256, pair([256, 4], [256, 4])), call(100, top([256, 5], [256, 5])), call(24, pair([24], [24, 1])), call(256, pair([256, 4], [1024]))],
        refused: [call(128, { entropy: ent, ...pair([3, 4], [256, 4]) }), call(128, pair([512], [1024])), call(128, pair([24], [24, 1])),
            call(128, pair([256, 4], [256, 3])), call(128, top([256, 4], [256, 5])), call(128, pair([256, 4], [24, 1])), call(128, { tokens: tensor([128], 'u32'), logprobs: tensor([128]) })],
    };
}

function fork() {
    const config = { nLayer: 2, nHead: 2, nKvHead: 1, nEmbd: 128, blockSize: 32 }, log = [];
    const context = (name) => ({ name, handle: {}, arena: () => ({ handle: {} }), sync: () => log.push(name) });
    const one = context('one'), two = context('two');
    const a = new q.KvCache(one, config), b = new q.KvCache(two, config), c = new q.KvCache(one, config);
    message(() => a.fork(b, 5));                               // ends at the library: no device
    const before = log.splice(0);
    message(() => a.fork(c, 5));
    const d = new q.KvCache(one, { ...config, nHead: 4, nKvHead: 2 });
    return { before, same: log, heads: message(() => a.fork(d, 3)) };
}

function trees() {
    const bad = [[-1, 4294967295], [-1, 4294967296], [-1, NaN], [-1, undefined], [-1, 0.7], [-1, null], [-1, '0'], [-1, 0n], [-1, , 0], [-1, -4294967296],
        Float64Array.from([-1, 0.5])];
    const { masks, depths } = q.treeMasks(Float32Array.from([-1, 0, 0, 1]));
    const p = new Int32Array([-1, 0]), m = new BigUint64Array(2), d = new Int32Array(2);
    return {
        refused: bad.map((b) => message(() => q.treeMasks(b))),
        kinds: [[Float32Array.from([-1, 0]), m, d], [p.buffer, m, d], [[-1, 0], m, d], [p, new Float64Array(2), d], [p, m, new Float32Array(2)], [p, m, new Uint32Array(2)]]
            .map((a) => message(() => q.addon.treeMasks(...a))),
        masks: Array.from(masks, String), depths: Array.from(depths),
    };
}

function table() {
    let syncs = 0;
    const model = Object.assign(Object.create(q.QuantLinearModel.prototype),
        { ctx: { handle: {}, sync: () => { syncs++; } }, weights: { handle: {}, size: 1 << 20 }, layout: new q.ArenaLayout(), f32Weights: new Map() });
    model.layout.take(256);
    const used = [model.layout.used];
    const long = message(() => model.makeRopeTable(1 << 20, 64, 1e4));
    used.push(model.layout.used);
    const bad = message(() => model.makeRopeTable(100, 64, 1e4));          // refused by the library: no handle
    used.push(model.layout.used);
    return { used, long, bad, syncs };
}

function read() {
    const from = { read: (offset, out) => out };
    return [undefined, 'f32', 'bytes', 'f16', 'u32', 'i32', 'u64'].map((dtype) => new q.Tensor(from, 0, 2, [2], dtype).read().constructor.name);
}

function addonExports() {
    const all = Object.getOwnPropertyNames(q.addon).filter((n) => typeof q.addon[n] === 'function').sort();
    return { all, hidden: all.filter((n) => !Object.keys(q.addon).includes(n)) };
}

function gpu() {
    const ctx = new q.Context(0);
    const model = new q.QuantLinearModel(ctx, 1 << 20), pool = new q.ActivationArena(ctx, 1 << 20);
    const x = pool.alloc([4, 20]), ids = pool.alloc([4, 2], 'i32'), tlp = pool.alloc([4, 2]);
    const logits = new Float32Array(80);
    for (let m = 0; m < 4; m++) { logits[20 * m + 2] = 5; logits[20 * m + 9] = 3; }
    x.write(logits);
    ids.write(new Int32Array(8).fill(-7));
    tlp.write(new Float32Array(8).fill(7));
    model.tokenLogprobs(x, 3, 20, { topIds: ids, topLogprobs: tlp });
    const i = ids.read(), l = tlp.read();
    const r = { ids: [0, 1, 2, 3].map((m) => Array.from(i.subarray(2 * m, 2 * m + 2))), behind: Array.from(l.subarray(6)) };
    pool.release();
    model.release();
    ctx.destroy();
    return r;
}

console.log(JSON.stringify({ widths, fork, trees, table, read, exports: addonExports, gpu }[process.argv[2]]()));
