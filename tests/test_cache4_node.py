"""The 4-bit key / value cache through the Node addon (web-engine_amd/node): its exports, its errors, and a decoding run that
equals the Python binding's byte for byte."""
import json
import pathlib
import shutil
import subprocess

import numpy as np
import pytest

import oracle_lib as O
import we

ROOT = pathlib.Path(__file__).resolve().parents[1]
NODE_DIR = ROOT / "web-engine_amd" / "node"
NODE = shutil.which("node")
pytestmark = pytest.mark.skipif(NODE is None or not (NODE_DIR / "we_node.node").exists(),
                                reason="node or the built addon (web-engine_amd/node/we_node.node) is missing")


def run(script, *args):
    out = subprocess.run([NODE, "-e", script, *args], cwd=NODE_DIR, capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr
    return json.loads(out.stdout.strip().splitlines()[-1])


def test_addon_exports_every_cache_function_and_throws_messages():
    names = {"we_cache4_" + n: "cache4" + n.capitalize() for n in ("bytes", "append", "load", "attention", "evict")}
    assert set(names) == set(we.header_functions(we.CACHE4_HEADER))
    got = run('const a = require("./we_node.node"); const r = {};'
              'for (const s of [[2, 4, 128, 64], [2, 4, 100, 64], [2, 4, 128, 65], [0, 4, 128, 64]]) '
              '{ try { r[s] = a.cache4Bytes(null, ...s); } catch (e) { r[s] = e.message; } }'
              'console.log(JSON.stringify({ keys: Object.keys(a), r, cls: typeof require("./index.js").Cache4 }));')
    assert set(names.values()) <= set(got["keys"]) and got["cls"] == "function"
    r = got["r"]
    assert r["2,4,128,64"] == 2 * 4 * 64 * 144
    assert r["2,4,100,64"] == "cache dim must be a multiple of 64 and at most 256, got 100"
    assert r["2,4,128,65"].startswith("cache capacity must be a multiple of 64") and "batch and kvHeads" in r["0,4,128,64"]


DRIVER = """
const fs = require("fs"), we = require("./index.js"), dir = process.argv[1];
(async () => {
  const graph = new we.Graph(0);
  const rd = (n) => graph.buffer(fs.readFileSync(`${dir}/${n}`));
  const c = new we.Cache4(graph, 2, 2, 128, 192);
  const counts = graph.buffer(new Int32Array([100, 71]));
  c.append(rd("k0"), rd("v0"), 100, we.BF16, { counts });
  const save = async (n, b) => fs.writeFileSync(`${dir}/${n}`, Buffer.from(await graph.read(b)));
  await save("y0", c.attention(rd("q0"), 100, 6, we.BF16, { counts, track: true }));
  c.evict(80, { sinks: 4, recent: 16 });
  c.append(rd("k1"), rd("v1"), 1, we.BF16);
  await save("y1", c.attention(rd("q1"), 1, 6, we.BF16, { maxLen: 96, track: true }));
  const kv = graph.buffer(2 * 3 * 2 * 128 * 2);
  c.load(null, kv, 3, we.BF16, { first: graph.buffer(new Int32Array([78, 69])) });
  await save("values", kv);
  for (const n of ["data", "lens", "seen", "pos", "weight"]) await save(n, c[n]);
  let message = "";
  try { c.attention(kv, 1, 3); } catch (e) { message = e.message; }
  let small = "";
  try { c.append(kv, kv, 90, we.BF16); } catch (e) { small = e.message; }
  c.free();
  graph.destroy();
  console.log(JSON.stringify({ message, small }));
})().catch((e) => { console.error(e); process.exit(1); });
"""


@pytest.mark.gpu
def test_node_decoding_equals_python(graph, tmp_path):
    rng = np.random.default_rng(0)
    data = {}
    for n, tokens in (("0", 100), ("1", 1)):
        for name, heads in (("q", 6), ("k", 2), ("v", 2)):
            x = rng.standard_normal(2 * tokens * heads * 128).astype(np.float32)
            data[name + n] = O.bf16_rne(x)
            (tmp_path / (name + n)).write_bytes(data[name + n].tobytes())
    said = run(DRIVER, str(tmp_path))
    assert said["message"] == "heads must be a multiple of kvHeads" and "k is too small" in said["small"]
    g, mark = graph, graph.mark()
    b = {k: g.buffer(v) for k, v in data.items()}
    c = we.Cache4(g, 2, 2, 128, 192)
    counts = g.buffer(np.array([100, 71], np.int32))
    c.append(b["k0"], b["v0"], 100, we.BF16, counts=counts)
    got = {"y0": c.attention(b["q0"], 100, 6, we.BF16, counts=counts, track=True)}
    c.evict(80, 4, 16)
    c.append(b["k1"], b["v1"], 1, we.BF16)
    got["y1"] = c.attention(b["q1"], 1, 6, we.BF16, max_len=96, track=True)
    got["values"] = g.buffer(2 * 3 * 2 * 128 * 2)
    g.cache4_load(c, 3, we.BF16, None, got["values"], first=g.buffer(np.array([78, 69], np.int32)), lens=c.lens)
    got.update({n: getattr(c, n) for n in ("data", "lens", "seen", "pos", "weight")})
    assert g.read(c.lens, dtype=np.int32).tolist() == [81, 72]
    for name, buf in got.items():
        assert (tmp_path / name).read_bytes() == g.read(buf).tobytes(), name
    g.release(mark)
