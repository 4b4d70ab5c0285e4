#!/bin/sh
# Builds the gfx950 HIP library (the C-ABI of include/uwc.h) into uwc_amd/libuwc_hip.so: every
# source compiled to an object in parallel, then one link. It needs hipcc alone ($HIPCC, by default ROCm's).
# Where python3 has torch, also the Python module uwc_amd/_kv.so; if that fails to compile, the library is
# built all the same and the script ends with an error.
#   -ffp-contract=off        no fused multiply-add: detrt's fp32 steps round once each
#   -packed-fp32-ops off     no v_pk_*_f32 from the compiler
set -e
cd "$(dirname "$0")"
OUT=../uwc_amd/libuwc_hip.so
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# the header's hash, which uwc_header_sha() returns and the Python binding checks at load
SHA=$(sha256sum ../../include/uwc.h | cut -c1-16)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-result -I../../include -DUWC_HEADER_SHA=\"$SHA\" ${UWC_HIPCC_EXTRA}"
TMP=$(mktemp -d)
trap 'rm -rf "$TMP"' EXIT
pids=""
# _kv.so, the Python module of uwc_kv_bind.cpp: host code over torch's headers, no GPU code
TORCH=$(python3 -c "import importlib.util as u, os; s = u.find_spec('torch'); print(os.path.dirname(s.origin) if s else '')" 2>/dev/null) || TORCH=""
bind=""
if [ -n "$TORCH" ]; then
  PYINC=$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")
  g++ -O2 -std=c++17 -fPIC -shared -D__HIP_PLATFORM_AMD__ -DUWC_HEADER_SHA="\"$SHA\"" -I../../include -I/opt/rocm/include \
    -isystem "$PYINC" -isystem "$TORCH/include" -isystem "$TORCH/include/torch/csrc/api/include" uwc_kv_bind.cpp \
    -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 -o "$TMP/_kv.so" &
  bind=$!
else
  rm -f ../uwc_amd/_kv.so
  echo "build.sh: python3 has no torch; the module _kv.so is left out" >&2
fi
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
if [ -n "$bind" ]; then
  if ! wait "$bind"; then
    rm -f ../uwc_amd/_kv.so
    echo "build.sh: the library is built, uwc_kv_bind.cpp failed to compile" >&2
    exit 1
  fi
  mv "$TMP/_kv.so" ../uwc_amd/_kv.so
fi
