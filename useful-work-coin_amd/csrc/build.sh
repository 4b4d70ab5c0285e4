#!/bin/sh
# Builds the gfx950 HIP library (the C-ABI of include/uwc.h) into uwc_amd/libuwc_hip.so: every
# source compiled to an object in parallel, then one link; and the Python module uwc_amd/_kv.so.
#   -ffp-contract=off        no fused multiply-add: detrt's fp32 steps round once each
#   -packed-fp32-ops off     no v_pk_*_f32 from the compiler
set -e
cd "$(dirname "$0")"
OUT=../uwc_amd/libuwc_hip.so
HIPCC=/opt/rocm/bin/hipcc
# the header's hash, which uwc_header_sha() returns and the Python binding checks at load
SHA=$(sha256sum ../../include/uwc.h | cut -c1-16)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-result -I../../include -DUWC_HEADER_SHA=\"$SHA\" ${UWC_HIPCC_EXTRA}"
TMP=$(mktemp -d)
trap 'rm -rf "$TMP"' EXIT
pids=""
# _kv.so, the Python module of uwc_kv_bind.cpp: host code over torch's headers, no GPU code
TORCH=$(python3 -c "import importlib.util as u, os; print(os.path.dirname(u.find_spec('torch').origin))")
PYINC=$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")
g++ -O2 -std=c++17 -fPIC -shared -D__HIP_PLATFORM_AMD__ -DUWC_HEADER_SHA="\"$SHA\"" -I../../include -I/opt/rocm/include \
  -isystem "$PYINC" -isystem "$TORCH/include" -isystem "$TORCH/include/torch/csrc/api/include" uwc_kv_bind.cpp \
  -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 -o "$TMP/_kv.so" &
pids="$pids $!"
for f in uwc_*.hip; do
  $HIPCC $FLAGS -c "$f" -o "$TMP/${f%.hip}.o" &
  pids="$pids $!"
done
fail=0
for p in $pids; do
  wait "$p" || fail=1
done
if [ "$fail" -ne 0 ]; then
  echo "build.sh: a source failed to compile" >&2
  exit 1
fi
$HIPCC --offload-arch=gfx950 -shared -fPIC "$TMP"/*.o -o "$OUT.tmp"
mv "$OUT.tmp" "$OUT"
mv "$TMP/_kv.so" ../uwc_amd/_kv.so
