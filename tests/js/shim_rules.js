'use strict';
// GPU run of createKvOps' calls with positions, rules, copies and drafts that
// stay: reads a case written by tests/test_gpu_js_rules.py, runs it through the
// addon, eagerly and recorded, and writes the results back.
const assert = require('assert');
const fs = require('fs');
const path = require('path');
const eff = require(path.join(__dirname, '..', '..', 'elffuss-engine_amd', 'js', 'index.js'));

async function main() {
  const dir = process.argv[2];
  const m = JSON.parse(fs.readFileSync(path.join(dir, 'meta.json'), 'utf8'));
  const device = await eff.requestDevice();
  const ops = eff.createQuantOps(device);
  const kv = eff.createKvOps(device, { ctx: ops.ctx });
  const sube = (name) => ops.upload(fs.readFileSync(path.join(dir, name + '.bin')), name);
  const rd = async (buf, n) => Array.from(new Float32Array(await eff.readback(device, buf, 0, n * 4)));
  const bytes = async (buf) => Array.from(new Uint8Array(await eff.readback(device, buf)));
  const out = {};

  const cache = kv.creaCache({ tipo: m.tipo, cabezas: m.cabezas, dim: m.dim, tokensPagina: m.pagina, paginas: m.paginas });
  device.queue.writeBuffer(cache.buf, 0, fs.readFileSync(path.join(dir, 'cache.bin')));
  const lote = { tabla: sube('table'), inicios: sube('starts'), largos: sube('lens'), secuencias: m.secuencias, tokens: m.tokens,
    paginasTabla: m.paginasTabla, maxNuevos: m.maxNuevos, maxLargo: m.maxLargo };
  const filas = { q: sube('q'), k: sube('k'), v: sube('v'), cabezasQ: m.cabezasQ, rope: kv.tablaRope(Float64Array.from(m.freqs), m.posiciones),
    posicionesRope: m.posiciones, dimRope: 2 * m.freqs.length };
  const giros = { en: sube('at'), ejes: m.ejes, eje: m.eje };
  const n = m.tokens * m.cabezasQ * m.dim;
  const q = await kv.anade(cache, lote, filas, giros);
  const reglas = { tope: m.tope, pendientes: sube('slopes'), arbol: sube('tree'), palabrasArbol: m.palabras };
  const y = await kv.atiende(cache, lote, q, m.cabezasQ, m.escala, { reglas });
  const z = await kv.atiende(cache, lote, q, m.cabezasQ, m.escala, { reglas: { rangos: sube('ranges') } });
  out.q = await rd(q, n);
  out.y = await rd(y, n);
  out.z = await rd(z, n);
  out.cache = await bytes(cache.buf);

  const g = await ops.ctx.grabaGrafo(async () => kv.atiende(cache, lote, await kv.anade(cache, lote, filas, giros), m.cabezasQ, m.escala, { reglas }));
  for (let i = 0; i < 3; i++) {
    device.queue.writeBuffer(g.salida, 0, new Float32Array(n).fill(7));
    g.lanza();
    assert.deepStrictEqual(await rd(g.salida, n), out.y);
  }
  g.destroy();

  const otra = kv.creaCache({ tipo: m.tipo, cabezas: m.cabezas, dim: m.dim, tokensPagina: m.pagina, paginas: m.paginas });
  device.queue.writeBuffer(otra.buf, 0, fs.readFileSync(path.join(dir, 'cache.bin')));
  const capas = [cache, otra], largos = sube('lens');
  await kv.copiaPaginas(capas, ops.upload(Uint32Array.from(m.copias), 'copias'), m.copias.length / 3);
  out.copied = [await bytes(cache.buf), await bytes(otra.buf)];
  await kv.conserva(capas, lote, sube('kept'), sube('counts'), largos);
  out.kept = [await bytes(cache.buf), await bytes(otra.buf)];
  out.lens = Array.from(new Uint32Array(await eff.readback(device, largos, 0, m.secuencias * 4)));
  await kv.conserva(capas, lote, sube('kept'), sube('counts'));

  const codigo = (f, c) => assert.throws(f, (e) => e.code === c);
  codigo(() => kv.anade(cache, lote, filas, { ...giros, ejes: 5 }), eff.STATUS.E_SHAPE);
  codigo(() => kv.anade(cache, lote, filas, { ...giros, ejes: 1 }), eff.STATUS.E_INVALID);
  codigo(() => kv.atiende(cache, lote, q, m.cabezasQ, 1, { reglas: { tope: -1 } }), eff.STATUS.E_INVALID);
  codigo(() => kv.atiende(cache, lote, q, m.cabezasQ, 1, { ventana: 1, reglas }), eff.STATUS.E_SHAPE);
  codigo(() => kv.copiaPaginas([cache, cache], largos, 1), eff.STATUS.E_INVALID);
  codigo(() => kv.copiaPaginas(capas, largos, 1000), eff.STATUS.E_BOUNDS);
  codigo(() => kv.conserva(capas, lote, lote.largos, lote.largos, lote.largos), eff.STATUS.E_INVALID);
  out.stats = device.stats();
  fs.writeFileSync(path.join(dir, 'out.json'), JSON.stringify(out));
  device.destroy();
}

main().catch((e) => { console.error(e); process.exit(1); });
