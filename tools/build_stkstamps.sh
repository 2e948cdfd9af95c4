#!/bin/bash
# dev: the persistent FFN stack with in-kernel stamps (-DSDH_STK_STAMPS) into tools/bin/variants/stkstamps/
set -e
cd "$(dirname "$0")/../llama.cpp_amd/csrc"
make -j8 2>&1 | grep -E "error|warning" || true
out=../../tools/bin/variants/stkstamps; mkdir -p $out
/opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops -DSDH_STK_STAMPS -c sdh_stack.hip -o $out/sdh_stack.o
objs=""; for o in build/*.o; do [ "$o" = "build/sdh_stack.o" ] || objs="$objs $o"; done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $out/libseeddelta_hip.so $objs $out/sdh_stack.o
echo built stkstamps
