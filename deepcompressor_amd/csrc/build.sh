#!/bin/bash
# Builds libdcq.so (gfx950 only) next to the package: deepcompressor_amd/libdcq.so
# -packed-fp32-ops: the two-value float32 instructions, which the compiler otherwise makes of ordinary code by itself,
# have given wrong results now and then (without them the bench kernels are as fast, to the spread between boxes).
# DCQ_REBUILD=1 compiles every file anew, else those that changed.
# -ffp-contract=off: the reference rounds after every multiply and add; a fused multiply-add changes results.
set -euo pipefail
HERE="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
ROOT="$(cd "$HERE/../.." && pwd)"
OUT="$HERE/../libdcq.so"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
FLAGS=(--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -fno-fast-math -I"$ROOT/include" -I"$HERE"
       -Xclang -target-feature -Xclang -packed-fp32-ops -Wall -Wno-unused-function -Wno-unused-variable ${DCQ_EXTRA_FLAGS:-})
OBJS=()
PIDS=()
mkdir -p "$HERE/build"
for src in "$HERE"/*.hip; do
  obj="$HERE/build/$(basename "${src%.hip}").o"
  if [[ -n "${DCQ_REBUILD:-}" || ! -f "$obj" || "$src" -nt "$obj" || "$HERE/build.sh" -nt "$obj" || "$HERE/dcq_common.cuh" -nt "$obj" || "$HERE/dcq_fp8.cuh" -nt "$obj" || "$ROOT/include/dcq.h" -nt "$obj" ]]; then
    rm -f "$obj"
    "$HIPCC" "${FLAGS[@]}" -c "$src" -o "$obj" &
    PIDS+=($!)
  fi
  OBJS+=("$obj")
done
for pid in "${PIDS[@]:-}"; do
  [[ -n "$pid" ]] && wait "$pid"
done
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$OUT" "${OBJS[@]}"
echo "built $OUT"
