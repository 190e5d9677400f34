'use strict';
/**
 * A copy of the Node host beside an addon folder without the addon of passes over many requests (tests/test_node_addons.py): what still runs, and what
 * is said where it is needed.
 *
 *   node addons_check.js <index.js of the copy>
 */
const q = require(process.argv[2]);

function message(fn) {
    try { fn(); return null; } catch (e) { return e.message; }
}
const ctx = { handle: {}, arena: (size) => ({ handle: {}, size, write() {} }) };
const config = { nLayer: 1, nHead: 6, nKvHead: 2, nEmbd: 384 };
const kv = new q.PagedKvCache(ctx, config, 4), pool = new q.ActivationArena(ctx, 1 << 20), a = kv.newSequence();
const batch = kv.batch(pool, [[a, 6]]);
const Q = pool.alloc([6, 384]), O = pool.alloc([6, 384]);
console.log(JSON.stringify({
    functions: Object.getOwnPropertyNames(q.addon).length, names: Object.keys(q).includes('batchAddon'), config: q.qwenKvDim(config),
    attend: message(() => kv.attend(0, Q, O, batch)), addon: message(() => q.batchAddon),
}));
