#!/bin/bash
# A/B builds of the library: scripts/build_variant.sh NAME SOURCE.hip REPLACES [extra compiler flags] -> exp/libtad_NAME.so
# (SOURCE.hip is compiled with the library's own flags in place of the object REPLACES, e.g. mm16)
# (the other objects are the ones of the regular build; select with TAD_HIP_LIB=exp/libtad_NAME.so)
set -e
cd "$(dirname "$0")/../timeautodiff_amd/csrc"
hipcc=${HIPCC:-/opt/rocm/bin/hipcc}
name=$1; src=$2; repl=$3; shift 3
mkdir -p ../../exp
obj=../../exp/${name}_$(basename ${src%.hip}).o
$hipcc $(make -s show-flags) -I. "$@" -c $src -o $obj
others=$(for f in $(make -s show-objects); do [ "$f" = "$repl.o" ] || echo $f; done)
$hipcc --offload-arch=gfx950 -shared -fPIC -o ../../exp/libtad_${name}.so $obj $others
echo built exp/libtad_${name}.so
