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
    for dep in "$src" "$HERE/build.sh" "$HERE"/*.h "$HERE/../../include/uresnet_hip.h"; do
        if [ ! -f "$obj" ] || [ "$dep" -nt "$obj" ]; then stale=1; fi
    done
    if [ "$stale" = 1 ]; then
        ( $HIPCC $FLAGS -c "$src" -o "$obj" ) &
        pids+=($!)
    fi
done
# the host module: host code against torch's headers, for the interpreter that will load it
PY="${PYTHON:-python3}"
HOST="$OUT/_host.so"
HOSTSRC=(module param_list gn_function)
TORCH="$($PY -c 'import importlib.util as u; print(u.find_spec("torch").submodule_search_locations[0])')"
PYINC="$($PY -c 'import sysconfig; print(sysconfig.get_paths()["include"])')"
for s in "${HOSTSRC[@]}"; do
    src="$HERE/host/$s.cpp"
    obj="$OBJ/host_$s.o"
    if [ ! -f "$obj" ] || [ "$src" -nt "$obj" ] || [ "$HERE/host/host.h" -nt "$obj" ] || [ "$HERE/build.sh" -nt "$obj" ] || [ "$HERE/../../include/uresnet_hip.h" -nt "$obj" ]; then
        ( "${CXX:-g++}" -O2 -std=c++17 -fPIC -Wall -D__HIP_PLATFORM_AMD__=1 -isystem "$TORCH/include" \
            -isystem "$TORCH/include/torch/csrc/api/include" -isystem "${ROCM_PATH:-/opt/rocm}/include" -I"$PYINC" -c "$src" -o "$obj" ) &
        pids+=($!)
    fi
done
for p in "${pids[@]:-}"; do [ -n "$p" ] && wait "$p"; done
objs=()
for s in "${SRCS[@]}"; do objs+=("$OBJ/$s.o"); done
$HIPCC --offload-arch=gfx950 -shared -fPIC -o "$OUT/liburesnet_hip.so" "${objs[@]}"
hobjs=()
for s in "${HOSTSRC[@]}"; do hobjs+=("$OBJ/host_$s.o"); done
"${CXX:-g++}" -shared -fPIC -o "$HOST" "${hobjs[@]}" -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10_hip -lc10 -Wl,-rpath,"$TORCH/lib"
echo "built $OUT/liburesnet_hip.so"
