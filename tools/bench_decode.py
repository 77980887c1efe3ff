"""Decode-only benchmark (MI355X): bench.py's two decode legs without the training step.
   python tools/bench_decode.py [repeats]      env: MGEN_DECODE_PARTS, MGEN_GEMM_SKINNY, LEGS=literal,long,short;
   MODEL=aria: the 650M Llama-style stand-in instead of the default decoder;
   KV=mxfp8 | mxfp4: that KV cache instead of bf16 (the fractions printed then count the bf16 cache's bytes);
   GREEDY=1 replaces the sampler by the argmax (what the step costs without the top-p search and the draw)"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "symbolic-music-generation_amd"))
sys.path.insert(0, ROOT)
import torch  # noqa: E402

import bench  # noqa: E402
from mgen import MidiLM, default_decoder, aria_style_llama  # noqa: E402

dev = torch.device("cuda:0")
cfg = aria_style_llama() if os.environ.get("MODEL") == "aria" else default_decoder()
model = MidiLM(cfg, device=dev, seed=0)
if os.environ.get("GREEDY") == "1":
    _generate = model.generate
    model.generate = lambda *a, **k: _generate(*a, **{**k, "do_sample": False})
KV = os.environ.get("KV", "bf16")
if KV != "bf16":
    _plain, _reserve = model.generate, model.reserve_kv_cache
    model.generate = lambda *a, **k: _plain(*a, **k, kv_cache=KV)
    model.reserve_kv_cache = lambda streams, length: _reserve(streams, length, kv_cache=KV)
for rep in range(int(sys.argv[1]) if len(sys.argv) > 1 else 1):
    legs = os.environ.get("LEGS", "literal,long").split(",")
    msg = []
    if "literal" in legs:
        a = bench.bench_decode(model, cfg, 256, 1, 4095, dev)
        msg.append(f"literal {a['ms_per_step']:.3f} ms/step frac {a['hbm_frac']:.4f}")
    if "long" in legs:
        b = bench.bench_decode(model, cfg, 256, 1792, 256, dev)
        msg.append(f"long context {b['ms_per_step']:.3f} frac {b['hbm_frac']:.4f}")
    if "short" in legs:
        c = bench.bench_decode(model, cfg, 256, 1, 512, dev)
        msg.append(f"contexts 1-512 {c['ms_per_step']:.3f} (host issue {model.last_decode_issue_s / 511 * 1e3:.3f} ms/step)")
    print(" | ".join(msg), flush=True)
