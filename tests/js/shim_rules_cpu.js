'use strict';
// CPU-only checks of createKvOps' positions, rules, copies and drafts that
// stay: what is no buffer or no number, and names that a description does not
// have, are errors before anything reaches a device (there is none here).
const assert = require('assert');
const path = require('path');
const eff = require(path.join(__dirname, '..', '..', 'elffuss-engine_amd', 'js', 'index.js'));
const { native } = eff;

const prestados = [];
const ctx = { alloc: (n) => { const b = { _h: {}, size: n }; prestados.push(b); return b; } };
const kv = eff.createKvOps({ _ctx: undefined }, { ctx });
const b = () => ({ _h: {} });
const muerto = { _h: {}, _alive: false };
const invalido = (f, re) => assert.throws(f, (e) => e.code === eff.STATUS.E_INVALID && re.test(e.message));
const cache = { tipo: 'F16', cabezas: 1, dim: 64, tokensPagina: 16, paginas: 1, buf: b() };
const lote = { tabla: b(), inicios: b(), largos: b(), secuencias: 1, tokens: 1, paginasTabla: 1, maxNuevos: 1, maxLargo: 1 };
const filas = { k: b(), v: b() };

for (const mal of [5, 'x', {}, muerto, true]) {
  invalido(() => kv.anade(cache, lote, filas, { en: mal }), /^en:/);
  for (const n of ['pendientes', 'rangos', 'arbol']) invalido(() => kv.atiende(cache, lote, b(), 1, 1, { reglas: { [n]: mal } }), new RegExp(`^${n}:`));
  invalido(() => kv.copiaPaginas([cache], mal, 1), /^copias:/);
  invalido(() => kv.copiaPaginas([{ ...cache, buf: mal }], b(), 1), /^buf:/);
  invalido(() => kv.conserva([cache], lote, mal, b()), /^guardados:/);
  invalido(() => kv.conserva([cache], lote, b(), mal), /^cuantos:/);
  invalido(() => kv.conserva([cache], lote, b(), b(), mal), /^largosNuevos:/);
}
for (const mal of [[4], [-1], [0.5], [300], ['1']]) invalido(() => kv.anade(cache, lote, filas, { en: b(), eje: mal }), /^eje:/);
invalido(() => kv.anade(cache, lote, filas, { en: b(), axis: [0] }), /«axis»/);
invalido(() => kv.anade(cache, lote, filas, { en: b(), ejes: 2 }), /varios ejes/);
invalido(() => kv.atiende(cache, lote, b(), 1, 1, { reglas: { cap: 5 } }), /«cap»/);
invalido(() => kv.copiaPaginas([cache], b()), /¿cuántas\?/);
// what is described rightly ends where these calls are switched off, with nothing lent
const apagado = (f) => assert.throws(f, (e) => e.code === eff.STATUS.E_DEVICE && /apagado/.test(e.message));
apagado(() => kv.anade(cache, lote, filas, { en: b(), ejes: 2, eje: [0, 1] }));
apagado(() => kv.atiende(cache, lote, b(), 1, 1, { reglas: { tope: 5, arbol: b(), palabrasArbol: 1 } }));
apagado(() => kv.copiaPaginas([cache], b(), 1));
apagado(() => kv.conserva([cache], lote, b(), b(), b()));
assert.strictEqual(prestados.length, 0);

for (const mal of [5, 'x', {}, true]) {
  invalido(() => native.kvAppend(undefined, {}, {}, {}, { at: mal }), /^at: not a buffer/);
  for (const n of ['slopes', 'ranges', 'tree']) invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, 1, 0, { [n]: mal }), new RegExp(`^${n}: not a buffer`));
  invalido(() => native.kvKeep(undefined, [{}], {}, undefined, undefined, mal), /^newLens: not a buffer/);
  invalido(() => native.kvCopy(undefined, [{ buf: mal }], undefined, 1), /^buf: not a buffer/);
}
for (const mal of [[0], new Uint16Array(2), new Uint8Array(129), 'x', 3]) invalido(() => native.kvAppend(undefined, {}, {}, {}, { axis: mal }), /^axis: not a Uint8Array/);
for (const mal of ['1', -1, 1.5, NaN, 2 ** 60, true, {}]) {
  invalido(() => native.kvAppend(undefined, {}, {}, {}, { axes: mal }), /^axes: not a whole number/);
  invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, 1, 0, { treeWords: mal }), /^treeWords: not a whole number/);
  invalido(() => native.kvCopy(undefined, [{}], undefined, mal), /^count: not a whole number/);
}
for (const mal of [undefined, {}, 5, new Uint8Array(4)]) {
  invalido(() => native.kvCopy(undefined, mal, undefined, 1), /^caches: not an array/);
  invalido(() => native.kvKeep(undefined, mal, {}, undefined, undefined), /^caches: not an array/);
}
invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, 1, 0, { cap: '5' }), /^cap: not a number/);
// what is left out goes on to the library, which has no context here
invalido(() => native.kvAppend(undefined, {}, {}, {}, {}), /elffuss_amd error/);
invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, 1, 0, {}), /elffuss_amd error/);
invalido(() => native.kvCopy(undefined, [], undefined, 0), /elffuss_amd error/);
invalido(() => native.kvKeep(undefined, [], {}, undefined, undefined), /elffuss_amd error/);
console.log('shim_rules_cpu ok');
