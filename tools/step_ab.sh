#!/bin/bash
# Same-box A/B of the training step: `bench.py` under different kernel switches (arguments: one quoted env list per run).
LOG=$(mktemp)
B="python bench.py --decode-tokens 0 --decode-full 0 --no-cpu-baseline --steps 8 --warmup 3"
for cfg in "$@"; do
  echo "== $cfg"
  env $cfg timeout -k 10 200 $B > $LOG 2>&1 || { tail -5 $LOG; exit 1; }
  python tools/show_bench.py $LOG | head -1
done
