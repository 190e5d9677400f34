'use strict';
/** Passes that the library always refuses, through the Node host's PagedKvCache (tests/test_batch_limits.py): message, and whether nothing was taken. */
const q = require('../../webllm_amd/js');

const base = { nLayer: 2, nHead: 6, nKvHead: 2, nEmbd: 384 };
const ctx = { handle: {}, arena: (size) => ({ handle: {}, size, write() {} }) };
const cache = (pages, config) => [new q.PagedKvCache(ctx, { ...base, ...config }, pages, 256, 'f16'), new q.ActivationArena(ctx, 1 << 24)];
const state = (kv) => JSON.stringify([kv.freePages, [...kv._lengths], [...kv._lists].map(([s, p]) => [s, p.length])]);
function refused(kv, pool, ...args) {
    const before = state(kv);
    try { kv.batch(pool, ...args); } catch (e) { return [e.message, state(kv) === before]; }
    return [null, false];
}
const out = { taken: [] };
{
    const [kv, pool] = cache(300), a = kv.newSequence(), b = kv.newSequence();
    out.rows = refused(kv, pool, [[a, 65000], [b, 536]]);
    out.padding = refused(kv, pool, [[a, 5]], 65536);
    out.none = refused(kv, pool, [[a, 0]], 0);
    out.taken.push(kv.batch(pool, [[a, 65000], [b, 535]]).M);
}
{
    const [kv, pool] = cache(300, { nHead: 128, nKvHead: 32, nEmbd: 128 * 64 }), a = kv.newSequence();
    out.wide = refused(kv, pool, [[a, 43691]]);
    out.taken.push(kv.batch(pool, [[a, 43690]]).M);
}
{
    const [kv, pool] = cache(5000), all = Array.from({ length: 4097 }, () => [kv.newSequence(), 1]);
    out.sequences = refused(kv, pool, all);
    out.taken.push(kv.batch(pool, all.slice(0, 4096)).desc.nSeq);
}
{
    const [kv, pool] = cache(5000, { nHead: 2048, nKvHead: 2048, nEmbd: 2048 * 16 }), all = Array.from({ length: 2049 }, (_, i) => [kv.newSequence(), i ? 0 : 1]);
    out.kvHeads = refused(kv, pool, all);
    out.taken.push(kv.batch(pool, all.slice(0, 2048)).desc.nSeq);
}
{
    const [kv, pool] = cache((1 << 18) + 2), a = kv.newSequence();
    kv._lists.set(a, Array.from({ length: 1 << 18 }, () => kv._take()));
    kv._lengths.set(a, (1 << 26) - 1);
    out.tokens = refused(kv, pool, [[a, 2]]);
    out.taken.push(kv.batch(pool, [[a, 1]]).desc.maxLen);
}
for (const [name, nHead, nKvHead, nEmbd] of [['head8', 4, 2, 32], ['head24', 4, 2, 96], ['head272', 2, 2, 544], ['headsApart', 4, 3, 64], ['heads8192', 8192, 8192, 8192 * 16]]) {
    try {
        cache(4, { nHead, nKvHead, nEmbd });
        out[name] = [null, false];
    } catch (e) { out[name] = [e.message, true]; }
}
console.log(JSON.stringify(out));
