#!/bin/bash
# build_variant_tu.sh <tu name without extension, e.g. elementwise> <out.so> [extra hipcc flags]:
# link a variant library that differs from the product only in ONE translation unit compiled with extra flags
cd "$(dirname "$0")/.."
TU=$1; shift
exec bash tools/build_variant.sh pivotcvae_amd/csrc/$TU.hip "$@"
