#!/bin/bash
# Build the gfx950 shared library in-tree: reid_gan_amd/libried_gan.so, and reid_gan_amd/_bind.so beside it.
#   ./build.sh       what changed since the last build: sources, flags, compilers, torch, Python
#   ./build.sh -f    everything
set -e
cd "$(dirname "$0")/reid_gan_amd/csrc"
OUT=../libried_gan.so
# (packed fp32 instructions stay off: some of their forms have given wrong results; the host pass does not know the feature)
FLAGS="-O3 --offload-arch=gfx950 -fPIC -std=c++17 -Wno-unused-result -Xclang -target-feature -Xclang -packed-fp32-ops"
BIND_FLAGS="-O2 -std=c++17 -fPIC -shared -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1"
[ "$1" = -f ] && rm -f *.o ../_bind.so
# What a built file was built with, beside its sources: objects of other flags or of another compiler are not linked
same() { [ -f "$1" ] && [ "$(cat "$1")" = "$2" ]; }
made="$FLAGS | $(hipcc --version)"
same hip.stamp "$made" || rm -f *.o
read -r T TV PV PY <<< "$(python3 -c "
import importlib.metadata as m, importlib.util as u, os, platform, sysconfig
print(os.path.dirname(u.find_spec('torch').origin), m.version('torch'), platform.python_version(), sysconfig.get_paths()['include'])")"
bound="$BIND_FLAGS | $(g++ --version) | $T $TV $PV $PY"
same bind.stamp "$bound" || rm -f ../_bind.so
rm -f hip.stamp bind.stamp
objs=()
pids=()
for f in api gemm elementwise special ssim loader legacy attn norm rotary xattn xattn_bwd adamw; do
  [ -f $f.hip ] || continue
  stale=0
  [ -f $f.o ] || stale=1
  for dep in $f.hip *.h ../../include/ried_gan.h; do
    [ $stale = 1 ] || { [ $dep -nt $f.o ] && stale=1; } || true
  done
  if [ $stale = 1 ]; then
    echo "hipcc $f.hip"
    rm -f $f.o
    hipcc $FLAGS -c $f.hip -o $f.o &
    pids+=($!)
  fi
  objs+=($f.o)
done
# the direct calls of the token operators (host code: torch tensors and autograd nodes in front of the C ABI)
if [ ! -f ../_bind.so ] || [ bind.cpp -nt ../_bind.so ] || [ ../../include/ried_gan.h -nt ../_bind.so ]; then
  echo "g++ bind.cpp"
  rm -f ../_bind.so
  g++ $BIND_FLAGS -I$T/include -I$T/include/torch/csrc/api/include -I$PY -I/opt/rocm/include bind.cpp -o ../_bind.so \
    -L$T/lib -lc10 -lc10_hip -ltorch_cpu -ltorch_python &
  pids+=($!)
fi
for p in "${pids[@]}"; do wait $p; done
hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT "${objs[@]}"
echo "$made" > hip.stamp
echo "$bound" > bind.stamp
echo "built $OUT"
