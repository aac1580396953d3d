#!/bin/bash
# a variant of the hot-path library with csrc/s2wino.hip (or SOURCE) compiled under extra flags, linked against the product's
# other objects (csrc/build/product/*.o):  tools/build_s2w_variant.sh NAME [SOURCE] [-D...]
set -e
cd "$(dirname "$0")/.."
name=$1; shift
C=swapping_autoencoder_pytorch_amd/csrc
src=$C/s2wino.hip
if [ -n "$1" ] && [ "${1#-}" = "$1" ]; then src=$1; shift; fi
others=$(ls $C/build/product/*.o | grep -v s2wino.hip.o)
mkdir -p tools/variants
/opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops -fPIC -Wno-unused-value -I include -I $C "$@" -c $src -o /tmp/s2w_$name.o
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC /tmp/s2w_$name.o $others -o tools/variants/$name.so
echo built tools/variants/$name.so
