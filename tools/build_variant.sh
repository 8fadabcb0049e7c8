#!/bin/bash
# build_variant.sh <source> <out.so> [extra hipcc flags]: link a variant library that differs from the product only in the translation
# unit of that name (before a "." or "_with_": catalog_bf16_with_pair_kernel.hip stands for catalog_bf16), compiled with extra flags.
# Flags and objects are the library's own (pivotcvae_amd/build.py), so build the library first.
set -e
SRC=$1; OUT=$2; shift 2
cd "$(dirname "$0")/.."
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
mkdir -p build/variants
OBJ=build/variants/$(basename $OUT .so).o
TU=$(basename $SRC .hip); TU=${TU%%_with_*}
FLAGS=$(python3 -c "from pivotcvae_amd import build; print(*build.FLAGS)")
OBJS=$(python3 -c "
import os, sys
from pivotcvae_amd import build
names = [os.path.splitext(s)[0] for s in build.SOURCES]
sys.argv[1] in names or sys.exit(f'no translation unit {sys.argv[1]}')
print(*[sys.argv[2] if n == sys.argv[1] else f'pivotcvae_amd/lib/obj/{n}.o' for n in names])" $TU $OBJ)
$HIPCC $FLAGS -I pivotcvae_amd/csrc "$@" -x hip -c $SRC -o $OBJ
$HIPCC --offload-arch=gfx950 -shared -fPIC -o $OUT $OBJS
echo built $OUT
