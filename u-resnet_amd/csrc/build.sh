#!/bin/bash
# Builds liburesnet_hip.so for gfx950 (MI355X) in-tree: u-resnet_amd/lib/liburesnet_hip.so
set -euo pipefail
HERE="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
OUT="$HERE/../lib"
OBJ="$HERE/../lib/obj"
mkdir -p "$OUT" "$OBJ"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# packed fp32 instructions off: some of their forms have given wrong results on this hardware (the host pass does not know
# the feature and says so; the warning is harmless)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops ${URESNET_EXTRA_FLAGS:-}"
SRCS=(common conv_igemm convt_gemm conv1x1_pw conv1x1_pw_wgrad conv3x3_tile conv3x3_wide wgrad3x3_tile conv_wgrad conv_group bn gnorm spatial loss optim adamw)
pids=()
for s in "${SRCS[@]}"; do
    src="$HERE/$s.hip"
    obj="$OBJ/$s.o"
    stale=0
    for dep in "$src" "$HERE"/*.h "$HERE/../../include/uresnet_hip.h"; do
        if [ ! -f "$obj" ] || [ "$dep" -nt "$obj" ]; then stale=1; fi
    done
    if [ "$stale" = 1 ]; then
        ( $HIPCC $FLAGS -c "$src" -o "$obj" ) &
        pids+=($!)
    fi
done
# the optimisers' parameter lists: host code against torch's headers, with the interpreter that will load it
PY="${PYTHON:-python3}"
LIST="$OUT/_param_list.so"
if [ ! -f "$LIST" ] || [ "$HERE/param_list.cpp" -nt "$LIST" ]; then
    (
        TORCH="$($PY -c 'import os, torch; print(os.path.dirname(torch.__file__))')"
        PYINC="$($PY -c 'import sysconfig; print(sysconfig.get_paths()["include"])')"
        ABI="$($PY -c 'import torch; print(int(torch._C._GLIBCXX_USE_CXX11_ABI))')"
        "${CXX:-g++}" -O2 -std=c++17 -fPIC -shared -Wall -D_GLIBCXX_USE_CXX11_ABI="$ABI" -isystem "$TORCH/include" \
            -isystem "$TORCH/include/torch/csrc/api/include" -I"$PYINC" "$HERE/param_list.cpp" -o "$LIST" \
            -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 -Wl,-rpath,"$TORCH/lib"
    ) &
    pids+=($!)
fi
for p in "${pids[@]:-}"; do [ -n "$p" ] && wait "$p"; done
objs=()
for s in "${SRCS[@]}"; do objs+=("$OBJ/$s.o"); done
$HIPCC --offload-arch=gfx950 -shared -fPIC -o "$OUT/liburesnet_hip.so" "${objs[@]}"
echo "built $OUT/liburesnet_hip.so"
