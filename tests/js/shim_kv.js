'use strict';
// GPU run of createKvOps and createLogitsOps: reads a case written by
// tests/test_gpu_js_kv.py, appends, attends and applies the rules through the
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
  const lg = eff.createLogitsOps(device, { ctx: ops.ctx });
  const sube = (name) => ops.upload(fs.readFileSync(path.join(dir, name + '.bin')), name);
  const rd = async (buf, n) => Array.from(new Float32Array(await eff.readback(device, buf, 0, n * 4)));
  const out = {};

  const cache = kv.creaCache({ tipo: m.tipo, cabezas: m.cabezas, dim: m.dim, tokensPagina: m.pagina, paginas: m.paginas });
  device.queue.writeBuffer(cache.buf, 0, fs.readFileSync(path.join(dir, 'cache.bin')));
  const lote = { tabla: sube('table'), inicios: sube('starts'), largos: sube('lens'), secuencias: m.secuencias, tokens: m.tokens,
    paginasTabla: m.paginasTabla, maxNuevos: m.maxNuevos, maxLargo: m.maxLargo };
  const rope = kv.tablaRope(Float64Array.from(m.freqs), m.maxLargo, 1);
  const fila = sube('rows');
  const qd = m.cabezasQ * m.dim, kd = m.cabezas * m.dim, paso = qd + 2 * kd;
  const filas = { q: fila, k: fila, v: fila, desdeK: qd, desdeV: qd + kd, pasoQ: paso, pasoK: paso, pasoV: paso, cabezasQ: m.cabezasQ,
    rope, posicionesRope: m.maxLargo, dimRope: 2 * m.freqs.length, modoRope: eff.ROPE.MITADES, normaQ: sube('qn'), normaK: sube('kn'),
    eps: 1e-5 };
  const q = await kv.anade(cache, lote, filas);
  const y = await kv.atiende(cache, lote, q, m.cabezasQ, m.escala, { ventana: m.ventana });
  out.q = await rd(q, m.tokens * qd);
  out.y = await rd(y, m.tokens * qd);
  out.cache = Array.from(new Uint8Array(await eff.readback(device, cache.buf)));

  // the same step recorded: the same bits
  const g = await ops.ctx.grabaGrafo(async () => {
    const q2 = await kv.anade(cache, lote, filas);
    return kv.atiende(cache, lote, q2, m.cabezasQ, m.escala, { ventana: m.ventana });
  });
  for (let i = 0; i < 3; i++) {
    device.queue.writeBuffer(g.salida, 0, new Float32Array(m.tokens * qd).fill(7));
    g.lanza();
    assert.deepStrictEqual(await rd(g.salida, m.tokens * qd), out.y);
  }
  g.destroy();

  const reglas = { historia: sube('history'), iniciosHistoria: sube('hstarts'), castigos: sube('pen'), idsSesgo: sube('bids'),
    valoresSesgo: sube('bvals'), iniciosSesgo: sube('bstarts'), mascara: sube('mask'), mascaraDe: sube('maskof'), mascaras: m.mascaras };
  const z = sube('logits');
  const l = await lg.aplica(z, m.filas, m.vocab, reglas);
  out.logits = Array.from(new Uint32Array(await eff.readback(device, l, 0, m.filas * m.vocab * 4)));
  assert.strictEqual(await lg.aplica(z, m.filas, m.vocab, reglas, { salida: z }), z);
  assert.deepStrictEqual(Array.from(new Uint32Array(await eff.readback(device, z, 0, m.filas * m.vocab * 4))), out.logits);

  // sample()'s penalties on the device: what sample() leaves in its Float32Array
  const v = new Float32Array(m.vocab).map((_, i) => Math.sin(i * 1.7) * 6);
  const ventana = [3, 9, 9, 400, 3, 77];
  const uno = { historia: ops.upload(Uint32Array.from(ventana), 'h'), iniciosHistoria: ops.upload(Uint32Array.from([0, 6]), 'hs'),
    castigos: ops.upload(Float64Array.from([1.1, 0, 0.3]), 'p') };
  const w = await lg.aplica(ops.upload(v, 'v'), 1, m.vocab, uno);
  const host = Float32Array.from(v);
  eff.sample(host, { previos: ventana, repeatPenalty: 1.1, presence: 0.3 });
  out.sampler = await rd(w, m.vocab);
  assert.deepStrictEqual(out.sampler, Array.from(host));

  assert.throws(() => kv.creaCache({ tipo: 'F8', cabezas: 1, dim: 64, tokensPagina: 16, paginas: 1 }), (e) => e.code === eff.STATUS.E_TYPE);
  assert.throws(() => kv.creaCache({ tipo: 'F16', cabezas: 1, dim: 65, tokensPagina: 16, paginas: 1 }), (e) => e.code === eff.STATUS.E_SHAPE);
  assert.throws(() => kv.atiende(cache, lote, q, m.cabezasQ + 1, 1), (e) => e.code === eff.STATUS.E_SHAPE);
  assert.throws(() => kv.anade(cache, Object.assign({}, lote, { maxLargo: 1 << 20 }), filas), (e) => e.code === eff.STATUS.E_BOUNDS);
  assert.throws(() => lg.aplica(z, m.filas + 1, m.vocab, reglas, { salida: z }), (e) => e.code === eff.STATUS.E_BOUNDS);
  out.stats = device.stats();
  fs.writeFileSync(path.join(dir, 'out.json'), JSON.stringify(out));
  device.destroy();
}

main().catch((e) => { console.error(e); process.exit(1); });
