# Builds the gfx950 shared library and the host-side checkers.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH  ?= gfx950
LIB   := mfcc_amd/lib/libmfcc_amd.so
SRC   := mfcc_amd/csrc/mfcc_amd.hip
SEQ   := mfcc_amd/csrc/sequence_ops.hip
SEQO  := build/sequence_ops.o
HDRS  := $(wildcard mfcc_amd/csrc/*.h) include/mfcc_amd.h
HIPFLAGS := --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -fno-signed-zeros -fno-slp-vectorize -Wall -Wno-unused-function
# the operators along time: no packed float32 instructions (some of their forms have given wrong results on this part), and no
# contraction of products and sums by the compiler, so that full and partial tiles round alike (fused where the source says fmaf)
SEQFLAGS := --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -c -fno-slp-vectorize -ffp-contract=off -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops

all: $(LIB) host_sim

$(SEQO): $(SEQ) mfcc_amd/csrc/sequence_kernels.h mfcc_amd/csrc/abi.h include/mfcc_amd.h
	@mkdir -p $(dir $@)
	$(HIPCC) $(SEQFLAGS) -o $@ $(SEQ)

build/mfcc_amd.o: $(SRC) $(HDRS)
	@mkdir -p $(dir $@)
	$(HIPCC) $(HIPFLAGS) -c -o $@ $(SRC)

$(LIB): build/mfcc_amd.o $(SEQO)
	@mkdir -p $(dir $@)
	$(HIPCC) --offload-arch=$(ARCH) -fPIC -shared -o $@ $^

host_sim: tests/host_sim/fft_sim tests/host_sim/libsequence_sim.so

tests/host_sim/fft_sim: tests/host_sim/fft_sim.cpp mfcc_amd/csrc/fft_lane.h mfcc_amd/csrc/tables.h
	g++ -O2 -std=c++17 -I mfcc_amd/csrc -o $@ $<

# the operators along time as host code (clang for its 16-bit types), for tests/test_sequence_kernels_cpu.py
HOSTCXX ?= /opt/rocm/llvm/bin/clang++
tests/host_sim/libsequence_sim.so: tests/host_sim/sequence_sim.cpp tests/host_sim/device/hip/hip_runtime.h $(SEQ) mfcc_amd/csrc/sequence_kernels.h mfcc_amd/csrc/abi.h include/mfcc_amd.h
	$(HOSTCXX) -x c++ -O1 -std=c++17 -fPIC -shared -ffp-contract=off -Wall -Wno-unused-function -I tests/host_sim/device -o $@ $<

# experimental builds for A/B timing: make variant NAME=noslp EXTRA="-fno-slp-vectorize"
variant: $(SRC) $(HDRS) $(SEQO)
	@mkdir -p build/variants
	$(HIPCC) $(HIPFLAGS) $(EXTRA) -c -o build/variants/$(NAME).o $(SRC)
	$(HIPCC) --offload-arch=$(ARCH) -fPIC -shared -o build/variants/libmfcc_$(NAME).so build/variants/$(NAME).o $(SEQO)

# the experimental eight-wave kernel (mfcc_amd/csrc/split_kernel.h) as a library of its own, for
# tools/split_check.py and tests/test_gpu_split_variant.py
split: build/variants/libmfcc_split.so
build/variants/libmfcc_split.so: $(SRC) $(HDRS) $(SEQO)
	@mkdir -p build/variants
	$(HIPCC) $(HIPFLAGS) -DMFCC_USE_SPLIT -c -o build/variants/split.o $(SRC)
	$(HIPCC) --offload-arch=$(ARCH) -fPIC -shared -o $@ build/variants/split.o $(SEQO)

asm: $(SRC) $(HDRS)
	@mkdir -p build
	$(HIPCC) --offload-arch=$(ARCH) -O3 -std=c++17 -fno-signed-zeros -fno-slp-vectorize $(EXTRA) -S --cuda-device-only -o build/mfcc_amd.s $(SRC) -Rpass-analysis=kernel-resource-usage 2> build/resource_usage.txt

clean:
	rm -rf mfcc_amd/lib build tests/host_sim/fft_sim tests/host_sim/libsequence_sim.so

.PHONY: all host_sim asm clean variant split
