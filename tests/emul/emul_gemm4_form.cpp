// Prints the form that the product of two MXFP4 operands takes for every line "M N K sms" of the input: "ks tn mt tiles".
#include <cstdio>

#include "../../jangq_b200/csrc/jq_mxfp4_form.cuh"

int main() {
    long long M, N, K, sms;
    while (std::scanf("%lld %lld %lld %lld", &M, &N, &K, &sms) == 4) {
        const jq::Gemm4Form f = jq::gemm4_form(M, N, K / 32, sms);
        std::printf("%d %d %lld %lld\n", f.ks, f.tn, (long long)f.mt, (long long)f.tiles);
    }
    return 0;
}
