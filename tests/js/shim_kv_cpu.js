'use strict';
// CPU-only checks of createKvOps and createLogitsOps: what is no buffer or no
// number, and names that a description does not have, are errors before
// anything reaches a device (there is none here).
const assert = require('assert');
const path = require('path');
const eff = require(path.join(__dirname, '..', '..', 'elffuss-engine_amd', 'js', 'index.js'));
const { native } = eff;

const prestados = [];
const ctx = { alloc: (n) => { const b = { _h: {}, size: n }; prestados.push(b); return b; } };
const device = { _ctx: undefined, createBuffer: (d) => ({ _h: {}, size: d.size }) };
const kv = eff.createKvOps(device, { ctx }), lg = eff.createLogitsOps(device, { ctx });
const b = () => ({ _h: {} });
const muerto = { _h: {}, _alive: false };
const invalido = (f, re) => assert.throws(f, (e) => e.code === eff.STATUS.E_INVALID && re.test(e.message));

// the host's layer: names and buffers, before a buffer is lent
const cache = { tipo: 'F16', cabezas: 1, dim: 64, tokensPagina: 16, paginas: 1, buf: b(), nota: 'a cache may carry more' };
const lote = { tabla: b(), inicios: b(), largos: b(), secuencias: 1, tokens: 1, paginasTabla: 1, maxNuevos: 1, maxLargo: 1 };
for (const mal of [5, 'normaK', {}, muerto, true]) {
  for (const nombre of ['normaK', 'normaQ', 'rope', 'q', 'k', 'v']) invalido(() => kv.anade(cache, lote, { k: b(), v: b(), [nombre]: mal }), new RegExp(`^${nombre}:`));
  for (const nombre of ['mascara', 'mascaraDe', 'historia', 'castigos', 'idsSesgo', 'valoresSesgo', 'iniciosSesgo', 'iniciosHistoria']) {
    invalido(() => lg.aplica(b(), 1, 64, { [nombre]: mal }), new RegExp(`^${nombre}:`));
  }
  for (const nombre of ['tabla', 'inicios', 'largos']) invalido(() => kv.anade(cache, { ...lote, [nombre]: mal }, { k: b(), v: b() }), new RegExp(`^${nombre}:`));
  invalido(() => kv.anade({ ...cache, buf: mal }, lote, { k: b(), v: b() }), /^buf:/);
  invalido(() => kv.atiende(cache, lote, mal, 1, 1), /^q:/);
  invalido(() => lg.aplica(mal, 1, 64, {}), /^logits:/);
}
invalido(() => kv.anade(cache, lote, { k: b(), v: b(), normak: b() }), /«normak»/);
invalido(() => kv.anade(cache, lote, { k: b(), v: b(), rope: b(), dimrope: 64 }), /«dimrope»/);
invalido(() => kv.atiende(cache, lote, b(), 1, 1, { window: 4 }), /«window»/);
invalido(() => lg.aplica(b(), 1, 64, { mascaras: 1, mask: b(), maskOf: b() }), /«mask»/);
invalido(() => lg.aplica(b(), 1, 64, {}, { stride: 64 }), /«stride»/);
assert.strictEqual(prestados.length, 0);

// the addon: what is there is a buffer, a whole number in its range, or a number
const filas = ['q', 'k', 'v', 'qOut', 'rope', 'qNorm', 'kNorm'], reglas = ['history', 'historyStarts', 'penalties', 'biasIds', 'biasValues',
  'biasStarts', 'mask', 'maskOf'];
for (const mal of [5, 'x', {}, true]) {
  for (const nombre of filas) invalido(() => native.kvAppend(undefined, {}, {}, { [nombre]: mal }), new RegExp(`^${nombre}: not a buffer`));
  for (const nombre of reglas) invalido(() => native.logitsApply(undefined, undefined, undefined, 1, 64, 0, { [nombre]: mal }), new RegExp(`^${nombre}: not a buffer`));
}
for (const mal of ['64', -1, 1.5, NaN, 2 ** 60, true, {}]) {
  const re = (n) => new RegExp(`^${n}: not a whole number`);
  for (const n of ['qOffset', 'vOffset', 'kStride', 'qHeads', 'ropeDim', 'ropeMode', 'ropePositions']) invalido(() => native.kvAppend(undefined, {}, {}, { [n]: mal }), re(n));
  for (const n of ['type', 'heads', 'headDim', 'pageTokens', 'pages']) invalido(() => native.kvAppend(undefined, { [n]: mal }, {}, {}), re(n));
  for (const n of ['seqs', 'tokens', 'tablePages', 'maxNew', 'maxLen']) invalido(() => native.kvAttn(undefined, {}, { [n]: mal }), re(n));
  invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, 1, mal), re('window'));
  invalido(() => native.logitsApply(undefined, undefined, undefined, 1, mal, 0, {}), re('vocab'));
  invalido(() => native.logitsApply(undefined, undefined, undefined, 1, 64, 0, { maskCount: mal }), re('maskCount'));
}
invalido(() => native.kvAppend(undefined, {}, {}, { normEps: '1e-5' }), /^normEps: not a number/);
invalido(() => native.kvAttn(undefined, {}, {}, undefined, 0, 0, undefined, 1, '1', 0), /^scale: not a number/);
// what is left out goes on to the library, which has no context here
invalido(() => native.kvAppend(undefined, {}, {}, { q: null, qNorm: undefined, ropeDim: null }), /elffuss_amd error/);
invalido(() => native.kvAttn(undefined, {}, {}, undefined, undefined, undefined, undefined, 1, 1), /elffuss_amd error/);
invalido(() => native.logitsApply(undefined, undefined, undefined, 1, 64, undefined, {}), /elffuss_amd error/);

// the rotation's frequencies are 64-bit numbers: the bytes of other arrays are not read as such
for (const mal of [new Float32Array(8), new Uint32Array(8), new Uint8Array(64), new ArrayBuffer(64), new DataView(new ArrayBuffer(64)), [1, 2], undefined]) {
  invalido(() => native.ropeTable(undefined, mal, 16, 1, undefined), /Float64Array/);
  invalido(() => kv.tablaRope(mal, 16), /Float64Array/);
}
for (const mal of ['16', -1, 0.5]) invalido(() => native.ropeTable(undefined, new Float64Array(4), mal, 1, undefined), /^positions:/);
invalido(() => native.ropeTable(undefined, new Float64Array(4), 16, '1', undefined), /^scale:/);
invalido(() => native.ropeTable(undefined, new Float64Array(4), 16, undefined, undefined), /elffuss_amd error/);
console.log('shim_kv_cpu ok');
