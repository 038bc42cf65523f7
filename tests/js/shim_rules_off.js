'use strict';
// GPU run of the calls with positions, rules, copies and drafts that stay, which
// this host has switched off: rightly described, through createKvOps and straight
// through the addon, they end in an error and launch nothing; the calls beside them run.
const assert = require('assert');
const path = require('path');
const eff = require(path.join(__dirname, '..', '..', 'elffuss-engine_amd', 'js', 'index.js'));
const { native } = eff;

async function main() {
  const device = await eff.requestDevice();
  const ops = eff.createQuantOps(device);
  const kv = eff.createKvOps(device, { ctx: ops.ctx });
  const u32 = (...x) => ops.upload(Uint32Array.from(x), 'u32');
  const filas1 = new Float32Array(64).fill(1);
  const cache = kv.creaCache({ tipo: 'F16', cabezas: 1, dim: 64, tokensPagina: 16, paginas: 3 });
  const lote = { tabla: u32(0), inicios: u32(0, 1), largos: u32(1), secuencias: 1, tokens: 1, paginasTabla: 1, maxNuevos: 1, maxLargo: 1 };
  const filas = { q: ops.upload(filas1, 'q'), k: ops.upload(filas1, 'k'), v: ops.upload(filas1, 'v'), cabezasQ: 1,
    rope: kv.tablaRope(Float64Array.from([1, 0.5]), 4), posicionesRope: 4, dimRope: 4 };
  const q = await kv.anade(cache, lote, filas);
  const y = await kv.atiende(cache, lote, q, 1, 1);
  const antes = device.stats();
  assert(!eff.KV_REGLAS_ENCENDIDO && antes.kvAppend === 1 && antes.kvAttn === 1);

  const apagado = (f) => assert.throws(f, (e) => e.code === eff.STATUS.E_DEVICE && /apagado|switched off/.test(e.message));
  apagado(() => kv.anade(cache, lote, filas, { en: u32(0) }));
  apagado(() => kv.atiende(cache, lote, q, 1, 1, { reglas: { tope: 5 } }));
  apagado(() => kv.copiaPaginas([cache], u32(0, 1, 16), 1));
  apagado(() => kv.conserva([cache], lote, u32(0), u32(1)));

  const c = { type: 1, heads: 1, headDim: 64, pageTokens: 16, pages: 3, buf: cache.buf._h };
  const b = { table: lote.tabla._h, starts: lote.inicios._h, lens: lote.largos._h, seqs: 1, tokens: 1, tablePages: 1, maxNew: 1, maxLen: 1 };
  const r = { q: filas.q._h, k: filas.k._h, v: filas.v._h, qHeads: 1, qOut: q._h, rope: filas.rope._h, ropePositions: 4, ropeDim: 4 };
  apagado(() => native.kvAppend(device._ctx, c, b, r, { at: u32(0)._h, axes: 1 }));
  apagado(() => native.kvAppend(device._ctx, c, b, r, { at: u32(0)._h, axes: 2, axis: Uint8Array.from([0, 1]) }));
  for (const reglas of [{ cap: 5 }, { slopes: filas.q._h }, { ranges: u32(0, 1)._h }, { tree: u32(1)._h, treeWords: 1 }, {}])
    apagado(() => native.kvAttn(device._ctx, c, b, q._h, 0, 0, y._h, 1, 1, 0, reglas));
  apagado(() => native.kvCopy(device._ctx, [c], u32(0, 1, 16)._h, 1));
  apagado(() => native.kvKeep(device._ctx, [c], b, u32(0)._h, u32(1)._h));
  apagado(() => native.kvKeep(device._ctx, [c], b, u32(0)._h, u32(1)._h, u32(0)._h));
  assert.deepStrictEqual(device.stats(), antes);

  native.kvAppend(device._ctx, c, b, r);
  native.kvAttn(device._ctx, c, b, q._h, 0, 0, y._h, 1, 1, 0);
  const got = new Float32Array(await eff.readback(device, y, 0, 256));
  assert(got.every((x) => x === 1));   // one token: its own value
  device.destroy();
  console.log('shim_rules_off ok');
}

main().catch((e) => { console.error(e); process.exit(1); });
