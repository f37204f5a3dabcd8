#!/bin/bash
# Builds a variant of libydet.so for A/B timing (tools/ab_conv.py):
#   tools/build_variant.sh <name> <conv|conv_pw|...> [<git rev> | -] [extra hipcc flags ...]
# -> tools/bin/libydet_<name>.so (that one source recompiled with the library's own flags and the extra ones, the other objects taken
# from build/csrc as they are).
set -e
cd "$(dirname "$0")/.."
name=$1; unit=$2; rev=${3:--}; shift; shift; shift || true
mkdir -p build/ab tools/bin
src=yolo_amd/csrc/$unit.hip
if [ "$rev" != "-" ]; then git show "$rev:yolo_amd/csrc/$unit.hip" > build/ab/${unit}_$name.hip; src=build/ab/${unit}_$name.hip; fi
flags=$(make -s --no-print-directory -C yolo_amd/csrc flags-$unit)
/opt/rocm/bin/hipcc $flags "$@" -c $src -o build/ab/${unit}_$name.o
objs=$(ls build/csrc/*.o | grep -v "/$unit.o")
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o tools/bin/libydet_$name.so build/ab/${unit}_$name.o $objs
echo built tools/bin/libydet_$name.so
